"""Trees that the tile kernel takes, and the bound of an output whose weights keep 16 bits."""
from __future__ import annotations

import numpy as np

from _paged_chosen import attend

# (q heads, kv heads, D, nodes, lengths, splits).  Automatic counts (splits 0) need enough to read; the number of
# columns a kv head, nodes x q heads / kv heads, picks the kernel: up to 64, 128, 256, and chunks of 256.
TILES = [
    # as the call plans itself: ranges cut anywhere, several sequences to a range and several ranges to a sequence
    (32, 8, 128, 16, (5200, 40, 0), 0),
    (32, 8, 128, 32, (2000, 1999, 3, 640), 0),
    (16, 4, 128, 64, (2600, 64, 1311), 0),
    (12, 4, 128, 133, (2500, 0), 0),
    (16, 4, 64, 14, (3100, 0, 1, 15, 16, 17, 63, 64, 65, 900, 1500, 31, 32, 33, 2048, 2047, 129, 7, 500, 1), 0),
    (32, 8, 64, 31, (1980, 1000, 0, 64, 128, 1919, 77, 5), 0),
    (32, 8, 64, 64, (1900, 1, 640, 1280), 0),
    (24, 8, 64, 100, (2200, 1100, 63), 0),
    # as many ranges as asked for: one a (sequence, kv head) of equal lengths, and others
    (8, 2, 128, 8, (130, 130), 1), (8, 2, 128, 30, (130, 130), 1), (8, 2, 128, 64, (130, 130), 1), (6, 2, 128, 90, (130, 130), 1),
    (8, 2, 64, 8, (130, 130), 1), (8, 2, 64, 30, (130, 130), 1), (8, 2, 64, 64, (130, 130), 1), (6, 2, 64, 90, (130, 130), 1),
    (8, 2, 128, 12, (900, 40, 0), 4), (8, 2, 128, 25, (700, 63, 1), 3), (8, 2, 128, 50, (640, 0, 65), 5), (8, 2, 128, 70, (300, 500), 2),
    (8, 2, 64, 12, (900, 40, 0), 4), (8, 2, 64, 25, (700, 63, 1), 3), (8, 2, 64, 50, (640, 0, 65), 5), (8, 2, 64, 70, (300, 500), 2),
]


def attend16(q, k, v, seen, out_bf16=True):
    """attend(), and the bound for weights of two bf16 terms: truncated and rounded, 2^-7 x 2^-8 of a weight are
    lost at most, and 2^-23 is added; then the result's own rounding."""
    out, w, err, _ = attend(q, k, v, seen, False, False)
    idx = np.flatnonzero(seen)
    err = err + (2.0 ** -15 + 2.0 ** -23) * (w[idx, None] * np.abs(v[idx])).sum(0)
    return out, err + 2.0 ** -8 * (np.abs(out) + err) if out_bf16 else err


def sees(capacity, length, bits):
    s = np.arange(capacity) < length
    s[length: length + bits.size] = bits
    return s


def formula(q, k, v, seen):
    """The formula in 64 bits with infinities and NaN as they are: q [D], k / v [L][D] of the tokens, seen bool [L]."""
    with np.errstate(invalid="ignore", over="ignore"):
        idx = np.flatnonzero(seen)
        s = k[idx].astype(np.float64) @ q.astype(np.float64) / np.sqrt(q.size)
        p = np.exp(s - s.max())
        p /= p.sum()
        return (p[:, None] * v[idx].astype(np.float64)).sum(0), p
