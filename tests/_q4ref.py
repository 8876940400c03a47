"""The 4-bit KV format and attention over it in 64 bits, from the format's
definition (include/operator_api.h), for the tests."""
from __future__ import annotations

import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def e4m3_values():
    """Value of every E4M3 byte (NaN for 0x7f, 0xff)."""
    b = np.arange(256)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * 2.0 ** (e - 7.0))
    v = np.where((b & 127) == 127, np.nan, v)
    return np.where(b > 127, -v, v)


E4M3 = e4m3_values()


def _nearest(x, table):
    """Index of the table value nearest to x >= 0 (saturating), ties to the even index."""
    mid = (table[1:] + table[:-1]) / 2
    lo = np.searchsorted(mid, x, side="left")    # a tie goes down
    hi = np.searchsorted(mid, x, side="right")   # a tie goes up
    return np.where(lo % 2 == 0, lo, hi)


def encode(x, pool_scale):
    """(codes [..., D], scale bytes [..., D / 16]) of fp16 rows x."""
    with np.errstate(over="ignore", invalid="ignore"):
        t = (x.astype(np.float32) / np.float32(pool_scale)).astype(np.float64)
    t = np.where(np.isnan(t), 0.0, t)
    g = t.reshape(t.shape[:-1] + (-1, 16))
    amax = np.abs(g).max(-1)
    sb = _nearest(np.minimum(amax / 6, 448.0), E4M3[:127])
    s = E4M3[sb][..., None]
    with np.errstate(invalid="ignore"):
        y = np.divide(np.abs(g), s, out=np.zeros_like(g), where=s > 0)
    c = _nearest(np.minimum(y, 6.0), LEVELS) | (np.signbit(g) * 8)
    c = np.where(s > 0, c, 0)
    return c.reshape(t.shape).astype(np.uint8), sb.astype(np.uint8)


def values(codes, sb, pool_scale):
    v = np.where(codes > 7, -LEVELS[codes & 7], LEVELS[codes & 7])
    s = E4M3[sb]
    return (v.reshape(v.shape[:-1] + (-1, 16)) * s[..., None]).reshape(v.shape) * float(
        np.float32(pool_scale))


def tile_index(D, is_key):
    """(byte, shift) [16, D] of every code and byte [16, D / 16] of every scale in a tile."""
    tok = np.arange(16)[:, None]
    d = np.arange(D)[None]
    if is_key:
        byte = tok * (D // 2) + (d % 16) // 4 * (D // 8) + d // 16 * 2 + d % 4 // 2
        sc = 8 * D + tok * (D // 16) + np.arange(D // 16)[None]
    else:
        byte = tok * (D // 2) + d // 2
        sc = 8 * D + np.arange(D // 16)[None] * 16 + tok
    return byte, 4 * (d % 2) + 0 * tok, sc


def unpack(pool, is_key):
    """(codes [nb, Hkv, bs, D], scale bytes [nb, Hkv, bs, D / 16]) of a pool."""
    nb, hkv, spp, tile = pool.shape
    D = tile // 9
    byte, shift, sc = tile_index(D, is_key)
    codes = (pool[..., byte] >> shift) & 15
    return codes.reshape(nb, hkv, 16 * spp, D), pool[..., sc].reshape(nb, hkv, 16 * spp, D // 16)


def pack(codes, sb, is_key):
    """Pool [nb, Hkv, bs / 16, 9 D] of codes [nb, Hkv, bs, D] and scale bytes."""
    nb, hkv, bs, D = codes.shape
    byte, shift, sc = tile_index(D, is_key)
    pool = np.zeros((nb, hkv, bs // 16, 9 * D), np.uint8)
    c = codes.reshape(nb, hkv, bs // 16, 16, D)
    for odd in (0, 1):
        pool[..., byte[:, odd::2]] |= (c[..., odd::2] << (4 * odd)).astype(np.uint8)
    pool[..., sc] = sb.reshape(nb, hkv, bs // 16, 16, D // 16)
    return pool


def attention(q, k, v, tables, lens, scale, num_blocks=None):
    """(out, bound) in 64 bits: q [B, Hq, D], pools as values [nb, Hkv, bs, D].
    Pages that the table does not name validly are masked. `bound` is what the
    kernel's arithmetic may be off by, element by element:
      scores are fp32 sums of exact products, D / 16 matrix steps of at most
      2^-22 of the sum of the terms' magnitudes each, plus the scaling's and
      the exponential's few units: a weight is off by exp(2 ds) - 1 at most;
      a weight is then rounded to fp16 (half a step: 2^-11 of it; where that is
      below fp16's normal range, half of 2^-24, 2^-32 of the largest weight,
      since the largest is at least 2^7), their products and sums are fp32
      (2^-22 a step and a tile), and the output is rounded to fp16 once
      (2^-11)."""
    q = q.astype(np.float64)
    B, Hq, D = q.shape
    nb, hkv, bs, _ = k.shape
    nb = nb if num_blocks is None else num_blocks
    out = np.zeros_like(q)
    bound = np.zeros_like(q)
    for b in range(B):
        n = int(np.clip(lens[b], 0, tables.shape[1] * bs))
        at = np.arange(n)
        page = tables[b, at // bs]
        ok = (page >= 0) & (page < nb)
        at, page = at[ok], page[ok]
        if not len(at):
            continue
        for h in range(hkv):
            kk, vv = k[page, h, at % bs], v[page, h, at % bs]
            for x in range(h * (Hq // hkv), (h + 1) * (Hq // hkv)):
                s = kk @ q[b, x] * scale
                mag = np.abs(kk) @ np.abs(q[b, x]) * abs(scale)
                p = np.exp(s - s.max())
                p /= p.sum()
                ds = (D / 16 + 4) * 2.0 ** -22 * mag.max() + 2.0 ** -20
                out[b, x] = p @ vv
                bound[b, x] = (p @ np.abs(vv)) * (
                np.expm1(2 * ds) + 2.0 ** -11 + (n / 16 + 16) * 2.0 ** -22)
            bound[b, x] += 2.0 ** -32 * p.max() * np.abs(vv).sum(0)
    return out, bound + 2.0 ** -11 * np.abs(out) + 2.0 ** -24
