"""A plain 64-bit statement of the 4-bit K/V cache (numpy): the block's rule, the
page layout byte by byte, and attention over what the pages hold."""
import numpy as np

NB = 32


def scale(m):
    """h of blocks whose value of largest magnitude is m (float64 array)."""
    t = np.clip(-m / 128, -508, 508)
    mant, e = np.frexp(t)  # |mant| in [0.5, 1): 7 bits are steps of 1/128
    r = np.ldexp(np.rint(mant * 128), e - 7)
    return np.rint(r * 2.0 ** 24) / 2.0 ** 24  # fp16 (subnormals below 2^-14)


def quantize(x):
    """(nibbles, h) of rows x [..., hdim] (fp32 or fp16 values, possibly not finite)."""
    x = np.asarray(x, np.float64)
    b = np.where(np.isnan(x), 0.0, x).reshape(*x.shape[:-1], -1, NB)
    top = np.abs(b).max(-1)
    m = np.where((b == -top[..., None]).any(-1), -top, top)
    h = scale(m)
    d = 16 * h[..., None]
    with np.errstate(all="ignore"):
        # limited before the floor: infinities stay ordered
        n = np.floor(np.clip(b / d, -100, 100) + 8.5)
    n = np.where(d == 0, 8, np.clip(np.where(np.isnan(n), 8, n), 0, 15))
    return n.astype(np.int64).reshape(x.shape), h


def held(x):
    """Rows as the cache holds them."""
    n, h = quantize(x)
    return ((n.reshape(*h.shape, NB) - 8) * (16 * h[..., None])).reshape(n.shape)


def page_bytes(kv, D, ps):
    return kv * ps * D * 9 // 16


def _k_nibble(D, i, e):
    byte = (i // 8 * 4 * D + i // 4 % 2 * 2 * D + e // 8 % 4 * (D // 2) + i % 4 * (D // 8)
            + e // 32 * 4 + e % 8 // 2)
    return byte, e % 2 + 0 * i


def _v_nibble(D, i, e):
    dt, full = e // 16, D // 64 * 4
    byte = i // 8 * 4 * D + i % 8 // 2 + np.where(
        dt < full, dt // 4 * 256 + e % 16 * 16 + dt % 4 * 4, full * 64 + e % 16 * 8 + (dt - full) * 4)
    return byte, i % 2 + 0 * e


def _scale_byte(D, ps, i, b):
    return ps * D // 2 + (i // 8 * (D // 32) + b) * 16 + (i % 4 * 2 + i // 4 % 2) * 2


def rows(pool, pages, pos, kv, D, ps, is_k):
    """Values [len(pos)][kv][D] of positions pos of a page list; pool uint8
    [npages][kv][ps * D * 9 / 16]."""
    pos = np.asarray(pos)
    pg = np.asarray(pages)[pos // ps]
    i, e = (pos % ps)[:, None], np.arange(D)[None, :]
    byte, odd = (_k_nibble if is_k else _v_nibble)(D, i, e)
    part = pool[pg]  # [n][kv][bytes]
    at = np.broadcast_to(byte[:, None, :], (len(pos), kv, D))
    v = np.take_along_axis(part, at, 2).astype(np.int64)
    n = (v >> (4 * odd[:, None, :])) & 15
    sb = _scale_byte(D, ps, i, np.arange(D // 32)[None, :])
    at = np.broadcast_to(sb[:, None, :], (len(pos), kv, D // 32))
    bits = (np.take_along_axis(part, at, 2).astype(np.uint16)
            | np.take_along_axis(part, at + 1, 2).astype(np.uint16) << 8)
    h = bits.view(np.float16).astype(np.float64)
    return (n - 8) * 16 * np.repeat(h, NB, axis=2)


def pack(values, kv, D, ps, is_k):
    """A pool (uint8 [npages][kv][bytes]) of rows values [npages * ps][kv][D]."""
    npages = len(values) // ps
    n, h = quantize(values)
    pool = np.zeros((npages, kv, ps * D * 9 // 16), np.uint8)
    i, e = np.arange(ps)[:, None], np.arange(D)[None, :]
    byte, odd = (_k_nibble if is_k else _v_nibble)(D, i, e)
    sb = _scale_byte(D, ps, i, np.arange(D // 32)[None, :])
    n = n.reshape(npages, ps, kv, D).transpose(0, 2, 1, 3)
    h = h.reshape(npages, ps, kv, D // NB).transpose(0, 2, 1, 3)
    for half in (0, 1):
        b, o = byte[odd == half], n[:, :, odd == half]
        pool[:, :, b] |= (o << (4 * half)).astype(np.uint8)
    bits = np.ascontiguousarray(h.astype(np.float16)).view(np.uint16)
    pool[:, :, sb] = bits & 255
    pool[:, :, sb + 1] = bits >> 8
    return pool


def rope(x, pos, cos, sin):
    """Rows x [n][heads][D] rotated at pos, each operation rounded to fp32."""
    H = x.shape[2] // 2
    c, s = cos[pos][:, None], sin[pos][:, None]
    a, b = x[..., :H], x[..., H:]
    return np.concatenate([a * c - b * s, b * c + a * s], -1).astype(np.float32)


def attend(q, k, v):
    """q [heads][D] over k, v [ctx][kv][D] in 64 bits; no position: zeros."""
    heads, D = q.shape
    out = np.zeros((heads, D))
    if len(k):
        G = heads // k.shape[1]
        for h in range(heads):
            t = k[:, h // G] @ q[h].astype(np.float64) / np.sqrt(D)
            p = np.exp(t - t.max())
            out[h] = p @ v[:, h // G] / p.sum()
    return out
