"""Plain forms, in numpy and 64 bits, of rotary positions, the 4-bit paged cache and attention over it."""
import math

import numpy as np

GROUP = 32


def turn(x, positions, rotary_dim, rates, half, magnitude=1.0):
    """x float64 [rows, heads, dim] -> turned."""
    y = x.copy()
    angle = positions.astype(np.float64)[:, None, None] * rates
    c, s = np.cos(angle) * magnitude, np.sin(angle) * magnitude
    n = rotary_dim
    first, second = (slice(0, n // 2), slice(n // 2, n)) if half else (slice(0, n, 2), slice(1, n, 2))
    y[..., first] = x[..., first] * c - x[..., second] * s
    y[..., second] = x[..., first] * s + x[..., second] * c
    return y


def rates(n, theta, scaling="none", factor=1.0, length=8192, low=1.0, high=4.0):
    out = []
    for i in range(n // 2):
        w = theta ** (-2.0 * i / n)
        if scaling == "linear":
            w /= factor
        elif scaling == "ntk":
            w = (theta * factor ** (n / (n - 2.0))) ** (-2.0 * i / n)
        elif scaling == "banded":
            b = min(1.0, max(0.0, (length * w / (2 * math.pi) - low) / (high - low)))
            w = b * w + (1 - b) * w / factor
        elif scaling == "yarn":
            index = lambda t: n * math.log(length / (t * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
            i0, i1 = max(0.0, math.floor(index(high))), min(n - 1.0, math.ceil(index(low)))
            b = 1 - min(1.0, max(0.0, (i - i0) / max(i1 - i0, 0.001)))
            w = b * w + (1 - b) * w / factor
        out.append(w)
    return np.array(out)


def quantise(x):
    """fp16 [..., dim] -> codes uint32 [..., dim], step and minimum fp16 [..., dim / 32]."""
    g = x.astype(np.float64).reshape(*x.shape[:-1], -1, GROUP)
    bad = ~np.isfinite(g).all(-1)
    g = np.where(bad[..., None], 0.0, g)
    low = g.min(-1)
    step = ((g.max(-1) - low) / 15.0).astype(np.float32).astype(np.float16)
    s = step.astype(np.float64)
    code = np.where(s[..., None] > 0, np.rint((g - low[..., None]) / np.where(s > 0, s, 1.0)[..., None]), 0.0).clip(0, 15)
    step, low = step.copy(), low.astype(np.float16)
    step[bad], low[bad] = np.nan, np.nan
    return code.astype(np.uint32).reshape(x.shape), step, low


def k_word_of(d, dim):
    p, r, q, w, b, a = d // 64, d // 32 % 2, d // 8 % 4, d // 4 % 2, d // 2 % 2, d % 2
    return q * (dim // 32) + 2 * p + w, 4 * (4 * a + 2 * b + r)


class Cache:
    """Host image of the four arrays."""

    def __init__(self, pages, page, heads, dim, rng=None):
        self.page, self.dim, self.n = page, dim, pages
        shapes = ((pages, heads, page, dim // 8), (pages, heads, dim // 32, page, 2), (pages, heads, page // 4, dim // 8, 4),
                  (pages, heads, dim // 32, page, 2))
        self.kc, self.ks, self.vc, self.vs = (np.zeros(s, np.uint16 if i % 2 else np.uint32) for i, s in enumerate(shapes))
        if rng is not None:  # garbage everywhere, NaN and infinities among the steps and minima
            for a in (self.kc, self.vc):
                a[...] = rng.integers(0, 2 ** 32, a.shape, dtype=np.uint64).astype(np.uint32)
            for a in (self.ks, self.vs):
                a[...] = rng.choice(np.array([0x7E00, 0x7C00, 0xFC00, 0x3C00, 0xFBFF], np.uint16), a.shape)

    def arrays(self):
        return self.kc, self.ks, self.vc, self.vs

    def put(self, page, slot, head, k, v):
        """One row (fp16 [dim]) of one head."""
        for which, x in (("k", k), ("v", v)):
            code, step, low = quantise(x)
            if which == "k":
                words = np.zeros(self.dim // 8, np.uint32)
                for d in range(self.dim):
                    at, shift = k_word_of(d, self.dim)
                    words[at] |= np.uint32(int(code[d]) << shift)
                self.kc[page, head, slot] = words
            else:
                nib = code.reshape(-1, 8)
                self.vc[page, head, slot // 4, :, slot % 4] = sum((nib[:, j].astype(np.uint32) << np.uint32(4 * j)) for j in range(8))
            s = self.ks if which == "k" else self.vs
            s[page, head, :, slot, 0] = step.view(np.uint16)
            s[page, head, :, slot, 1] = low.view(np.uint16)

    def rows(self, which, page, slots, head):
        """float64 [len(slots), dim] of what the cache stands for."""
        s = (self.ks if which == "k" else self.vs)[page, head][:, slots].view(np.float16).astype(np.float64)  # [groups, n, 2]
        if which == "k":
            at, shift = np.array([k_word_of(d, self.dim) for d in range(self.dim)]).T
            code = self.kc[page, head][slots][:, at] >> shift.astype(np.uint32) & 15
        else:
            d = np.arange(self.dim)
            code = self.vc[page, head][slots // 4][:, d // 8, :][np.arange(len(slots)), :, slots % 4] >> (4 * (d % 8)).astype(np.uint32) & 15
        with np.errstate(invalid="ignore", over="ignore"):
            return np.repeat(s[..., 1], GROUP, 0).T + np.repeat(s[..., 0], GROUP, 0).T * code

    def sequence(self, which, table, count, head):
        """float64 [count, dim] of positions 0..count-1, and which of them have a page."""
        out, there = np.zeros((count, self.dim)), np.zeros(count, bool)
        for j in range(-(-count // self.page)):
            t = np.arange(j * self.page, min(count, (j + 1) * self.page))
            if j < len(table) and 0 <= table[j] < self.n:
                out[t] = self.rows(which, table[j], t - j * self.page, head)
                there[t] = True
        return out, there


def attend(cache, q, starts, lengths, table, scale, window, max_query=None, max_length=None):
    """q fp16 [rows, heads, dim] -> (result float64, sum p |v|, largest scale sum |q k| over seen positions); rows without a
    sequence are NaN in the result."""
    rows, heads, dim = q.shape
    kv = cache.kc.shape[1]
    out, size, reach = np.full(q.shape, np.nan), np.zeros(q.shape), np.zeros((rows, heads))
    x = q.astype(np.float64)
    capacity = min(table.shape[1] * cache.page, max_length or 1 << 40)
    for b in range(len(lengths)):
        n = starts[b + 1] - starts[b]
        if n <= 0:
            continue
        seen_all = max(0, min(int(lengths[b]), capacity))
        for h in range(kv):
            keys, there = cache.sequence("k", table[b], seen_all, h)
            vals, _ = cache.sequence("v", table[b], seen_all, h)
            for i in range(n if max_query is None else min(n, max_query)):
                r, pos = starts[b] + i, int(lengths[b]) - n + i
                t = np.arange(seen_all)
                see = there & (t <= pos) & ((t > pos - window) if window else True)
                for g in range(heads // kv):
                    head = h * (heads // kv) + g
                    if not see.any():
                        out[r, head] = 0
                        continue
                    with np.errstate(invalid="ignore", over="ignore"):
                        s = keys[see] @ x[r, head] * scale
                        p = np.exp(s - s.max())
                        p /= p.sum()
                        out[r, head] = p @ vals[see]
                        size[r, head] = p @ np.abs(vals[see])
                        reach[r, head] = (np.abs(keys[see]) @ np.abs(x[r, head])).max() * abs(scale)
    return out, size, reach
