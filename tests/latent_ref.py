"""The latent cache, the attention over it and rotary positions in 64 bits (numpy), for the tests."""
import math

import numpy as np
import torch


def values():
    """What the 256 E4M3 bytes stand for: sign, 4 bits of exponent (bias 7), 3 of fraction; 127 and 255 are NaN."""
    v = np.empty(256)
    for u in range(128):
        e, f = u >> 3, u & 7
        v[u] = f * 2.0 ** -9 if e == 0 else (8 + f) * 2.0 ** (e - 10)
    v[127] = np.nan
    v[128:] = -v[:128]
    return v


VALUES = values()
FINITE = VALUES[:127]                 # ascending from 0 to 448


def codes_of(x):
    """The E4M3 bytes nearest x, ties to the even byte; |x| past 448 gives 448, NaN gives 127."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.where(np.isnan(x), 0, np.abs(x)), 448)
    hi = np.clip(np.searchsorted(FINITE, a), 1, 126)
    lo = hi - 1
    mid = (FINITE[lo] + FINITE[hi]) / 2
    c = np.where(a < mid, lo, np.where(a > mid, hi, np.where(lo % 2 == 0, lo, hi)))
    return np.where(np.isnan(x), 127, c + 128 * np.signbit(x)).astype(np.uint8)


def same_codes(a, b):
    """Equal bytes, a NaN's sign and a zero's aside."""
    a, b = VALUES[a], VALUES[b]
    return bool(((a == b) | (np.isnan(a) & np.isnan(b))).all())


def scale_of(amax):
    if amax == 0:
        return 2.0 ** -32
    e = math.floor(math.log2(amax / 448)) - 1
    while 448 * 2.0 ** e < amax:
        e += 1
    return 2.0 ** max(-32, min(32, e))


class Cache:
    """A cache's codes and scales on the host, and append on it."""

    def __init__(self, cache):
        self.page, self.pages = cache.page, cache.pages
        self.codes = [cache.c_codes.cpu().numpy().copy(), cache.r_codes.cpu().numpy().copy()]
        self.scales = cache.scales.cpu().numpy().astype(np.float64)

    def append(self, xs, table, lens, counts):
        row = 0
        for t, n, k in zip(table, lens, counts):
            for j in range(max(n - k, 0) // self.page, -(-min(n, len(t) * self.page) // self.page)):
                lo, hi = max(n - k, j * self.page, 0), min(n, (j + 1) * self.page)
                p = t[j]
                if hi > lo and 0 <= p < self.pages:
                    for part, x in enumerate(xs):
                        new = np.asarray(x[row + lo - (n - k):row + hi - (n - k)], np.float64)
                        scale = scale_of(np.abs(np.where(np.isfinite(new), new, 0)).max())
                        codes, off = self.codes[part][p], lo - j * self.page
                        if off > 0:
                            scale = max(scale, self.scales[p, part])
                            if scale != self.scales[p, part]:
                                codes[:off] = codes_of(VALUES[codes[:off]] * (self.scales[p, part] / scale))
                        codes[off:hi - j * self.page] = codes_of(np.where(np.isfinite(new), new / scale, np.nan))
                        self.scales[p, part] = scale
            row += k

    def tokens(self, t, n):
        """(latents, rotary keys, whether there is such a token) of a sequence's first n tokens."""
        pos = np.arange(min(n, len(t) * self.page))
        p = np.asarray(t, np.int64)[pos // self.page]
        there = (p >= 0) & (p < self.pages)
        p = np.where(there, p, 0)
        return [VALUES[self.codes[i][p, pos % self.page]] * self.scales[p, i, None] for i in (0, 1)] + [there]


def attend(cache, q, table, lens, counts, scale):
    """(out, lse, the size of what is summed per output value: sum p |c|, and of the scores: scale sum |q k|)."""
    T, H, _ = q.shape
    d_c = cache.codes[0].shape[2]
    out, size = np.zeros((T, H, d_c)), np.zeros((T, H, d_c))
    lse, spread = np.full((T, H), -np.inf), np.zeros((T, H))
    row = 0
    for t, n, k in zip(table, lens, counts):
        c, r, there = cache.tokens(t, max(n, 0))
        for i in range(k):
            sees = min(max(max(n, 0) - k + i + 1, 0), len(c))
            ci, ri, at = c[:sees][there[:sees]], r[:sees][there[:sees]], row + i
            if len(ci):
                s = scale * (q[at, :, :d_c] @ ci.T + q[at, :, d_c:] @ ri.T)
                spread[at] = abs(scale) * (np.abs(q[at, :, :d_c]) @ np.abs(ci).T + np.abs(q[at, :, d_c:]) @ np.abs(ri).T).max(1)
                m = s.max(1, keepdims=True)
                e = np.exp(s - m)
                total = e.sum(1, keepdims=True)
                out[at], size[at] = (e / total) @ ci, (e / total) @ np.abs(ci)
                lse[at] = (m + np.log(total))[:, 0]
        row += k
    return out, lse, size, spread


def rope(x, positions, inv_freq, scale, layout, start):
    """x [T, heads, width] float64 turned; (result, the size of each turned value: scale (|a| + |b|))."""
    n = 2 * len(inv_freq)
    # the turn in 64 bits, less its whole part in Python's integers where a product has more bits than that
    turns = np.array([[math.fmod(float(p) * f, 2 * math.pi) for f in inv_freq] for p in positions])
    c, s = scale * np.cos(turns)[:, None], scale * np.sin(turns)[:, None]
    part = x[..., start:start + n]
    a, b = (part[..., :n // 2], part[..., n // 2:]) if layout == "half" else (part[..., 0::2], part[..., 1::2])
    u, v, w = a * c - b * s, b * c + a * s, abs(scale) * (np.abs(a) + np.abs(b))
    join = (lambda p, q: np.stack([p, q], -1).reshape(part.shape)) if layout == "interleaved" else (lambda p, q: np.concatenate([p, q], -1))
    y, size = x.copy(), np.zeros_like(x)
    y[..., start:start + n], size[..., start:start + n] = join(u, v), join(w, w)
    return y, size


def pool(lens, page, gen, spare=3, extra=0):
    """(table as lists of equal length, pages): a shuffled pool's pages for sequences of these lengths."""
    used = [-(-max(n, 0) // page) for n in lens]
    pages = sum(used) + spare
    order = torch.randperm(pages, generator=gen).tolist()
    width, table, at = max(1, *used) + extra, [], 0
    for u in used:
        table.append(order[at:at + u] + [-1] * (width - u))
        at += u
    return table, pages
