"""Page bounds and page selection in 64 bits, from their definitions
(include/operator_api.h), for the tests."""
from __future__ import annotations

import numpy as np


def tame(x, dtype):
    big = float(np.finfo(dtype).max)
    return np.nan_to_num(x.astype(np.float64), nan=0.0, posinf=big, neginf=-big)


def bounds(k, tables, lens, num_new, into, dtype):
    """Bounds [nb, Hkv, 2, D] after a call: `into` with the due pages' entries
    replaced. k: pool values [nb, Hkv, bs, D] (any type)."""
    nb, hkv, bs, D = k.shape
    out = into.copy()
    for b, n in enumerate(np.clip(lens, 0, tables.shape[1] * bs)):
        first = max(0, n - num_new) // bs if num_new else 0
        for at in range(first, -(-n // bs)):
            page = tables[b, at]
            if 0 <= page < nb:
                x = tame(k[page, :, :min(bs, n - at * bs)], dtype)
                out[page, :, 0] = x.min(1).astype(dtype)
                out[page, :, 1] = x.max(1).astype(dtype)
    return out


def select(q, bnd, tables, lens, bs, keep, sink, recent, scale, num_blocks):
    """Kept pages [B, Hkv, keep], ascending, -1 past the last."""
    B, Hq, D = q.shape
    hkv = bnd.shape[1]
    qq = tame(q, q.dtype) * np.sign(scale)
    out = np.full((B, hkv, keep), -1, np.int32)
    for b in range(B):
        n = -(-int(np.clip(lens[b], 0, tables.shape[1] * bs)) // bs)
        page = tables[b, :n]
        ok = (page >= 0) & (page < num_blocks)
        for h in range(hkv):
            if n <= keep:
                kept = np.nonzero(ok)[0]
            else:
                bd = bnd[np.where(ok, page, 0), h].astype(np.float64)
                g = qq[b, h * (Hq // hkv):(h + 1) * (Hq // hkv)]
                score = (np.maximum(g, 0) @ bd[:, 1].T + np.minimum(g, 0) @ bd[:, 0].T).max(0)
                must = (np.arange(n) < sink) | (np.arange(n) >= n - recent)
                rest = np.nonzero(ok & ~must)[0]
                rest = rest[np.argsort(-score[rest], kind="stable")][:keep - sink - recent]
                kept = np.sort(np.concatenate([np.nonzero(must & ok)[0], rest]))
            out[b, h, :len(kept)] = kept
    return out
