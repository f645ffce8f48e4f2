"""CPU oracle of the quantised K/V cache and the attention over it, in numpy.

Codes and scales are computed as include/nuq.h defines them (float32 up to the
code, as a stored byte has one right answer); attention is float64 throughout.
Tiles are addressed value by value, from the layout's formulas alone."""
import numpy as np

OFFSET = {4: 8, 8: 128}


def geometry(bits, d):
    """chunk bytes, units, codes bytes of a plane, tile bytes"""
    chunk = min(16, d * bits // 32)
    return chunk, d * bits // 32 // chunk, 2 * d * bits, d * (4 * bits + 2)


def bf16(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)


def quantise(bits, x):
    """x [..., D] finite float32 -> integer codes (no offset) and float16 scales [..., D / 32]."""
    g = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, 32)
    high, low = g.max(-1), g.min(-1)
    if bits == 4:
        m = np.where(high >= -low, high, low)
        d = bf16(np.clip(m * np.float32(-0.125), np.float32(-2720), np.float32(2720))).astype(np.float16)
    else:
        u = (np.maximum(high, -low) / np.float32(127)).view(np.uint32).astype(np.uint64)
        up = ((u + 0xFFFFF) & 0xFFF00000).astype(np.uint32).view(np.float32)
        d = np.minimum(up, np.float32(56)).astype(np.float16)
    wide = d.astype(np.float32)[..., None]
    q = np.where(wide == 0, np.float32(0), np.rint(g / np.where(wide == 0, np.float32(1), wide)))
    q = np.clip(q, -8, 7) if bits == 4 else np.clip(q, -127, 127)
    return q.astype(np.int32).reshape(x.shape), d


def stored(bits, k, v):
    """What the cache holds after k, v [..., D]: float64 values and the poison flag [...] (NaN throughout)."""
    bad = ~(np.isfinite(k).all(-1) & np.isfinite(v).all(-1))
    out = []
    for x in (k, v):
        q, d = quantise(bits, np.where(bad[..., None], np.float32(0), x).astype(np.float32))
        value = (q.reshape(*d.shape, 32) * d.astype(np.float64)[..., None]).reshape(x.shape)
        out.append(np.where(bad[..., None], np.nan, value))
    return out[0], out[1], bad


def k_place(bits, d, token, dim):
    """(byte, bit) of a K code and byte of its scale in a tile."""
    chunk, units, codes, _ = geometry(bits, d)
    wide = d // units
    u, g, h, e = dim // wide, dim % wide // 32, dim % 32 // 8, dim % 8
    at = ((u * 16 + token) * 4 + h) * chunk + g * bits
    scale = codes + 2 * (token * (d // 32) + dim // 32)
    if bits == 8:
        return at + e, 0, scale
    bit = 4 * (e // 2) + 16 * (e % 2)
    return at + bit // 8, bit % 8, scale


def v_place(bits, d, token, dim):
    chunk, units, codes, _ = geometry(bits, d)
    wide = d // units
    per = wide // 16
    u, n, j = dim // wide, dim % wide // per, dim % per
    at = codes + d + (((u * 4 + token // 4) * 16 + n) * 4 + token % 4) * (chunk // 4)
    scale = 2 * codes + d + 2 * ((token // 4 * (d // 32) + dim // 32) * 4 + token % 4)
    return (at + j, 0, scale) if bits == 8 else (at + j // 2, 4 * (j % 2), scale)


def tile_values(bits, d, tile, place):
    """float64 [16, D] of one tile's bytes."""
    out = np.empty((16, d))
    for t in range(16):
        for c in range(d):
            byte, bit, scale = place(bits, d, t, c)
            code = int(tile[byte]) >> bit & ((1 << bits) - 1)
            out[t, c] = (code - OFFSET[bits]) * float(np.frombuffer(tile[scale:scale + 2].tobytes(), np.float16)[0])
    return out


def attention(q, k, v, position, group, scale, window=0, absent=None):
    """q [n][heads][D] at positions position .. position + n - 1; k, v
    [length][kv heads][D] (float64, NaN where poisoned); absent [length]: on no
    page. Returns o, sum p|v|, sum over the visible |v|, largest sum |q k| scale a row."""
    n, heads, d = q.shape
    o = np.zeros((n, heads, d))
    mass, plain = np.zeros_like(o), np.zeros_like(o)
    reach = np.zeros((n, heads))
    for i in range(n):
        p = position + i
        if p < 0:
            continue
        first = max(0, p - window + 1) if window else 0
        see = np.arange(first, min(p + 1, len(k)))
        if absent is not None:
            see = see[~absent[see]]
        if len(see) == 0:
            continue
        for h in range(heads):
            kk, vv = k[see, h // group], v[see, h // group]
            s = kk @ q[i, h].astype(np.float64) * scale
            reach[i, h] = np.max(np.abs(kk) @ np.abs(q[i, h].astype(np.float64))) * scale
            w = np.exp(s - s.max())
            w /= w.sum()
            o[i, h], mass[i, h], plain[i, h] = w @ vv, w @ np.abs(vv), np.abs(vv).sum(0)
    return o, mass, plain, reach
