"""Plain forms of a step over a paged cache held in 8 bits, on the host: the cache's codes and scales bit for bit
(numpy fp32, whose division is IEEE's), pages and slots in Python integers, attention and rotary positions in float64
with bounds on what fp32 kernels may be off."""
from __future__ import annotations

import numpy as np
import torch

MOST = {"int8": np.float32(127), "fp8": np.float32(448)}
E4M3 = torch.arange(256, dtype=torch.int16).to(torch.uint8).view(torch.float8_e4m3fn).float().numpy()


def decode(codes, kind):
    """Values (fp32, before the scale) of stored bytes."""
    codes = np.ascontiguousarray(codes)
    return codes.view(np.int8).astype(np.float32) if kind == "int8" else E4M3[codes.view(np.uint8)]


def encode(y, kind):
    """Bytes of quotients y (fp32): nearest code, ties to even, cut to the largest."""
    y = np.asarray(y, np.float32)
    if kind == "int8":
        return np.clip(np.rint(y), -127, 127).astype(np.int8).view(np.uint8)
    mag = np.minimum(np.abs(y.astype(np.float64)), 448.0)
    table = E4M3[:127].astype(np.float64)
    hi = np.searchsorted(table, mag)                       # table[hi - 1] < mag <= table[hi]
    lo = np.maximum(hi - 1, 0)
    up, down = table[hi] - mag, mag - table[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return (code | np.where(np.signbit(y), 128, 0)).astype(np.uint8)


def code_under(x, scale, kind):
    x, scale = np.asarray(x, np.float32), np.float32(scale)
    if not scale > 0:
        return np.zeros(x.shape, np.uint8)
    with np.errstate(all="ignore"):
        return encode(x / scale, kind)


class Cache:
    """Codes [page][Hkv][2][page_tokens][D] (K, then V) and scales [page][Hkv][2]."""

    def __init__(self, pages, heads, pt, d, kind):
        self.kind, self.pt, self.heads, self.d, self.pages = kind, pt, heads, d, pages
        self.codes = np.zeros((pages, heads, 2, pt, d), np.uint8)
        self.scales = np.zeros((pages, heads, 2), np.float32)

    def append(self, keys, values, slots):
        """Rows [T][Hkv][D] at their slots, a run of a page at a time."""
        t = 0
        while t < len(slots):
            s = int(slots[t])
            n = 1
            if 0 <= s < self.pages * self.pt:
                while t + n < len(slots) and s % self.pt + n < self.pt and slots[t + n] == s + n:
                    n += 1
                for h in range(self.heads):
                    for w, x in ((0, keys), (1, values)):
                        self._run(s // self.pt, s % self.pt, h, w, np.asarray(x[t:t + n, h], np.float32))
            t += n

    def _run(self, page, off, h, w, x):
        codes, most = self.codes[page, h, w], MOST[self.kind]
        old = np.float32(0) if off == 0 else self.scales[page, h, w]
        new = np.abs(x).max() / most if np.isfinite(x).all() else np.float32(np.nan)
        scale = old if np.isnan(old) or old >= new else new
        if off and scale > old:
            codes[:off] = code_under(decode(codes[:off], self.kind) * old, scale, self.kind)
        codes[off:off + len(x)] = code_under(x, scale, self.kind)
        self.scales[page, h, w] = scale

    def tokens(self, table, length):
        """K and V [Hkv][length][D] (float64) of a sequence."""
        n = -(-length // self.pt)
        got = []
        for w in (0, 1):
            v = decode(self.codes[table[:n], :, w], self.kind).astype(np.float64) * self.scales[table[:n], :, w][..., None, None]
            got.append(v.transpose(1, 0, 2, 3).reshape(self.heads, -1, self.d)[:, :length])
        return got

    def upload(self, cache):
        """Into a QuantizedKVCache's pools."""
        k = np.ascontiguousarray(self.codes[:, :, 0])
        v = np.ascontiguousarray(self.codes[:, :, 1].transpose(0, 1, 3, 2))
        for pool, x in ((cache.k_pool, k), (cache.v_pool, v)):
            pool.view(torch.int8).copy_(torch.from_numpy(x.view(np.int8)))
        cache.scales.copy_(torch.from_numpy(self.scales))


def download(cache):
    """A QuantizedKVCache's codes and scales in Cache's layout."""
    k = cache.k_pool.view(torch.int8).cpu().numpy().view(np.uint8)
    v = cache.v_pool.view(torch.int8).cpu().numpy().view(np.uint8).transpose(0, 1, 3, 2)
    return np.stack((k, v), 2), cache.scales.cpu().numpy()


# ---------------------------------------------------------------- pages and slots
class Pages:
    """Lengths, tables and the free list, sequence by sequence."""

    def __init__(self, batch, per, pages, pt):
        self.batch, self.per, self.pages, self.pt = batch, per, pages, pt
        self.lens, self.table = [0] * batch, [[-1] * per for _ in range(batch)]
        self.stack, self.count = list(range(pages)), pages

    def step(self, counts, room, keep=None):
        """(starts, positions, slots) of a step."""
        pt, of = self.pt, lambda n: -(-n // self.pt)
        if keep is not None:
            for b in range(self.batch):
                kept = min(max(int(keep[b]), 0), self.lens[b])
                for p in range(of(self.lens[b]) - 1, of(kept) - 1, -1):
                    self.stack[self.count], self.table[b][p] = self.table[b][p], -1
                    self.count += 1
                self.lens[b] = kept
        have, asked, rows, starts, positions, slots = self.count, 0, 0, [0], [], []
        for b in range(self.batch):
            n, at = max(int(counts[b]), 0), self.lens[b]
            if at + n > self.per * pt:
                n = 0
            need = of(at + n) - of(at)
            asked, rows = asked + need, rows + n
            if (need and asked > have) or rows > room:
                n = need = 0
            for p in range(of(at), of(at) + need):
                self.count -= 1
                self.table[b][p] = self.stack[self.count]
            for pos in range(at, at + n):
                positions.append(pos)
                slots.append(self.table[b][pos // pt] * pt + pos % pt)
            self.lens[b] = at + n
            starts.append(starts[-1] + n)
        pad = [-1] * (room - len(slots))
        return starts, positions + pad, slots + pad


# ---------------------------------------------------------------- rotary positions
def rotate64(x, positions, inv_freq, magnitude, interleaved):
    """Rows [T][heads][D] (float64) turned, and what |x| contributes to each value (for bounds)."""
    x = np.asarray(x, np.float64)
    n = len(inv_freq)
    a = np.asarray(positions, np.float64)[:, None, None] * np.asarray(inv_freq, np.float64)
    c, s = np.cos(a) * magnitude, np.sin(a) * magnitude
    i = (np.arange(0, 2 * n, 2), np.arange(1, 2 * n, 2)) if interleaved else (np.arange(n), np.arange(n, 2 * n))
    y, size = x.copy(), np.zeros_like(x)
    p, q = x[..., i[0]], x[..., i[1]]
    y[..., i[0]], y[..., i[1]] = p * c - q * s, q * c + p * s
    size[..., i[0]] = size[..., i[1]] = (np.abs(p) + np.abs(q)) * abs(magnitude)
    return y, size


# ---------------------------------------------------------------- attention
def attend64(q, k, v, length, scale, wide):
    """Newest rows q [R][Hq][D] (float64) over k, v [Hkv][L][D] (float64): out and how far fp32 arithmetic may be off,
    before the output's own rounding.  wide: softmax weights of 24 bits instead of 16."""
    rows, hq, d = q.shape
    heads, group = k.shape[0], hq // k.shape[0]
    out, off = np.full(q.shape, np.nan), np.full(q.shape, np.nan)
    u = 2.0 ** -24
    end = np.repeat(length - rows + 1 + np.arange(rows), group)          # tokens that a column sees
    live = end > 0
    if not live.any():
        return out, off
    hidden = np.arange(length)[None] >= end[live][:, None]
    for h in range(heads):
        qq = q[:, h * group: (h + 1) * group].reshape(rows * group, d)[live]
        with np.errstate(all="ignore"):
            x = np.where(hidden, -np.inf, qq @ k[h].T * scale)
            m = x.max(1, keepdims=True)
            p = np.exp(x - m)
            p /= p.sum(1, keepdims=True)
            o = p @ v[h]
            # sums over 3 D terms, each product exact; three products with scales and log2 e; the difference from
            # the largest score; exp2 to 2 ulp
            seen = np.where(hidden, 0.0, x)
            e = (3 * d + 8) * u * (np.abs(qq) @ np.abs(k[h]).T) * scale + 4 * u * np.abs(seen)
            e = np.where(hidden, 0.0, e)
            e = e + e.max(1, keepdims=True) + u * np.abs(seen - m) * 2 + 4 * u
            sums = (end[live][:, None] + 16) * u
            weight = (4 * u if wide else 2.0 ** -15) + sums
            bound = (p * e) @ np.abs(v[h]) + (p @ np.abs(v[h])) * weight + np.abs(o) * ((p * e).sum(1, keepdims=True) + sums + u)
        for target, value in ((out, o), (off, bound)):
            full = np.full((rows * group, d), np.nan)
            full[live] = value
            target[:, h * group: (h + 1) * group] = full.reshape(rows, group, d)
    return out, off


def close(got, want, off, rounding):
    """got (float64) is within off and a rounding of want; NaN where want is, and nowhere else."""
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan), (np.isnan(got) != nan).sum()
    worst = np.abs(got - want)[~nan] / (off[~nan] + np.abs(want[~nan]) * rounding + 1e-37)
    assert worst.size == 0 or worst.max() <= 1.0, worst.max()


HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}   # half a step of the type
