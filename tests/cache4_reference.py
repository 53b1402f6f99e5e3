"""The 4-bit cache and attention in 64 bits, for the tests (numpy)."""

from __future__ import annotations

import numpy as np

CODES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)


def encode(x):
    """(codes uint8 [..., D / 2], scale bytes [..., D / 32]) of rows x [..., D], by distance to every code."""
    blocks = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 32)
    top = np.abs(blocks).max(-1)
    finite = np.isfinite(top)
    _, e = np.frexp(np.where(finite, top, 1.0))
    byte = np.where(top > 0, np.maximum(e - 1 - 2 + 127, 1), 1)
    byte = np.where(finite, byte, 255)
    a = np.abs(np.where(finite[..., None], blocks, 0.0)) / np.exp2(np.where(finite, byte, 127) - 127.0)[..., None]
    d = np.abs(a[..., None] - CODES)
    best = d.min(-1, keepdims=True)
    tied = d == best  # of two codes at one distance the even one
    code = np.where(tied & (np.arange(8) % 2 == 0), np.arange(8), np.where(tied, np.arange(8) + 100, 200)).min(-1)
    code = np.where(code >= 100, code - 100, code)
    code = code + 8 * (np.signbit(blocks) & finite[..., None])
    code = code.reshape(*x.shape[:-1], -1, 2).astype(np.uint8)
    return code[..., 0] | code[..., 1] << 4, byte.astype(np.uint8)


def decode(codes, scales):
    """Rows [..., D] in 64 bits."""
    c = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    v = np.where(c >= 8, -1.0, 1.0) * CODES[c & 7]
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127.0))
    return (v.reshape(*v.shape[:-1], -1, 32) * s[..., None]).reshape(v.shape)


def attend(q, K, V, allowed, scaling):
    """(out, bound) of queries [R, D] over rows [N, D] with allowed [R, N].  bound: sum p |v| (2 delta + N 2^-24), the
    part of the error that fp32 scores and sums may have: a score's products and sum are within delta = (D + 4) 2^-24
    sum |q k| s of it (and its exponential's argument within 3 2^-24 of the largest score), so a weight within
    2 delta after division, and a sum of N terms within N 2^-24."""
    out, bound = np.zeros((len(q), V.shape[1])), np.zeros((len(q), V.shape[1]))
    for r in range(len(q)):
        n = np.flatnonzero(allowed[r])
        if len(n) == 0:
            continue
        k, v = K[n], V[n]
        s = k @ q[r] * scaling
        p = np.exp(s - s.max())
        p /= p.sum()
        out[r] = p @ v
        delta = 2.0 ** -24 * ((len(q[r]) + 4) * (np.abs(k) @ np.abs(q[r])).max() * scaling + 3 * np.abs(s).max())
        bound[r] = p @ np.abs(v) * (2 * delta + (len(n) + 16) * 2.0 ** -24)
    return out, bound
