"""A ragged step over pages in plain numpy: page lists and slot maps, and attention with a
window and sinks in 64 bits."""
import numpy as np


def tables(have, add, held, pages, ring, free, page, window, sinks, max_rows):
    """si_kv_step's outputs (pages and ring as copies), by its description."""
    pages, ring = pages.copy(), ring.copy()
    nseq, max_pages = pages.shape
    npages, (begin, count) = ring.size, (int(x) for x in free)
    kept = -(-sinks // page)
    out = dict(start=[0], taken=[0], ctx=[], held=[], seq=[], pos=[], slot=[])
    back, moves, code = [], [], 0
    for i in range(nseq):
        h, a, t, g = int(have[i]), max(int(add[i]), 0), int(held[i][0]), int(held[i][1])
        if h < 0:
            back += [pages[i, j] for j in range(t) if j < kept or j >= kept + g]
            out["ctx"].append(0)
            out["held"].append((0, 0))
        elif h + a > max_pages * page or h > t * page:
            code |= 4
            out["ctx"].append(h)
            out["held"].append((t, g))
        else:
            now = g
            while kept + now < t and (kept + now + 1) * page <= h - window + 1:
                back.append(pages[i, kept + now])
                now += 1
            more = max(0, -(-(h + a) // page) - t)
            moves += [(i, t + k) for k in range(more)]
            out["seq"] += [i] * a
            out["pos"] += range(h, h + a)
            out["ctx"].append(h + a)
            out["held"].append((t + more, now))
        out["start"].append(len(out["seq"]))
        out["taken"].append(len(moves))
    rows, took = len(out["seq"]), len(moves)
    code |= (rows > max_rows) | 2 * (took > count)
    if code:
        out = dict(start=[0] * (nseq + 1), taken=[0] * (nseq + 1),
                   ctx=[max(int(h), 0) for h in have], held=[tuple(x) for x in held], seq=[],
                   pos=[], slot=[])
        free, status = (begin, count), (code, rows, took, 0)
    else:
        for k, (i, j) in enumerate(moves):
            pages[i, j] = ring[(begin + k) % npages]
        for k, x in enumerate(back):
            ring[(begin + count + k) % npages] = x
        out["slot"] = [int(pages[i, p // page]) * page + p % page
                       for i, p in zip(out["seq"], out["pos"])]
        free = ((begin + took) % npages, count - took + len(back))
        status = (0, rows, took, len(back))
    for k in ("seq", "pos", "slot"):
        out[k] = np.array(list(out[k]) + [-1] * (max_rows - len(out[k])), np.int64)
    for k in ("start", "taken", "ctx"):
        out[k] = np.array(out[k], np.int64)
    return dict(out, held=np.array(out["held"], np.int64).reshape(nseq, 2), pages=pages, ring=ring,
                free=np.array(free), status=np.array(status))


def visible(p, window, sinks):
    """The positions that a row at position p sees, as an array."""
    t = np.arange(p + 1)
    return t[(t > p - window) | (t < sinks)]


def attend(q, k, v, p, window, sinks, per):
    """(out, bound) of one row q [qheads][D] at position p over rows k, v [L][kvheads][D]:
    its outputs in 64 bits, and how far 32-bit ones may be.

    The bound: a score is a sum of D products in 32 bits, of q to 22 bits (as two fp16
    halves), off by (D + 8) 2^-24 of the sum of its terms' sizes S at most, so a weight by
    twice that (both of its quotient's sides) relative; a weight is held to 22 bits, the
    exponential and the sums over n positions round n + 16 times, each by 2^-24 of the sum of
    the |w v|."""
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    if p < 0:
        return out, bound
    t = visible(p, window, sinks)
    D = q.shape[1]
    for h in range(q.shape[0]):
        kk, vv = k[t, h // per].astype(np.float64), v[t, h // per].astype(np.float64)
        x = q[h].astype(np.float64)
        with np.errstate(invalid="ignore", over="ignore"):
            s = kk @ x / np.sqrt(D)
            w = np.exp(s - s.max())
            w /= w.sum()
            out[h] = w @ vv
            S = (np.abs(kk) @ np.abs(x)).max() / np.sqrt(D)
            bound[h] = 2.0 ** -24 * (4 * (D + 8) * S + 2 * t.size + 64) * (w @ np.abs(vv))
    return out, bound
