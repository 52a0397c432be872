"""The 8-bit cache, attention over it, eviction and rotary positions from their definitions, in
numpy and 64 bits, a sequence and a head at a time: what the GPU tests compare with."""
import math

import numpy as np

BLOCK = 16


def _codes(form):
    """Every value that a code can have, ascending, and whether its last bit is even."""
    if form == "int8":
        v = np.arange(-127, 128)
        return v.astype(np.float64), v % 2 == 0
    values = {}
    for code in range(127):      # 127 is NaN
        e, m = code >> 3, code & 7
        values[code] = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
    pos = [(v, c % 2 == 0) for c, v in values.items()]
    both = sorted([(-v, even) for v, even in pos if v] + pos)
    return np.array([v for v, _ in both]), np.array([even for _, even in both])


CODES = {form: _codes(form) for form in ("e4m3", "int8")}
MOST = {"e4m3": 448.0, "int8": 127.0}


def nearest(x, form):
    """The code nearest to each x (in units of the scale), ties to the even one; beyond the last: the last."""
    values, even = CODES[form]
    x = np.asarray(x, dtype=np.float64)
    nan = np.isnan(x)
    x = np.where(nan, 0.0, x)
    hi = np.clip(np.searchsorted(values, x), 1, len(values) - 1)
    lo = hi - 1
    to_lo, to_hi = x - values[lo], values[hi] - x
    pick = np.where(to_lo < to_hi, lo, np.where(to_lo > to_hi, hi, np.where(even[lo], lo, hi)))
    out = values[pick]
    return np.where(nan, np.nan if form == "e4m3" else 0.0, out)


def scale_for(top, form):
    """The smallest power of two, 2^-126 or more, with which `top` is at most the largest code."""
    s = 2.0 ** -126
    while top > MOST[form] * s:
        s *= 2.0
    return s


def hold(x):
    """What an append sees of its rows."""
    x = np.asarray(x, dtype=np.float64)
    return np.where(np.isnan(x), x, np.clip(x, -2.0 ** 127, 2.0 ** 127))


class Cache:
    """[slots][kv_heads][capacity][head_dim] values as codes times scales."""

    def __init__(self, slots, kv_heads, head_dim, capacity, form):
        self.form, self.capacity = form, capacity
        self.codes = np.zeros((2, slots, kv_heads, capacity, head_dim))
        self.scales = np.zeros((2, slots, kv_heads, capacity // BLOCK))
        self.weights = np.zeros((slots, kv_heads, capacity), dtype=np.float32)

    def append(self, slot, position, rows):
        """rows: (keys, values), [n, kv_heads, head_dim] each."""
        n = rows[0].shape[0]
        for side in range(2):
            x = hold(rows[side])
            for h in range(self.codes.shape[2]):
                for b in range(self.capacity // BLOCK):
                    new = [r for r in range(b * BLOCK, (b + 1) * BLOCK) if max(position, 0) <= r < position + n]
                    if not new:
                        continue
                    v = x[[r - position for r in new], h]
                    mags = np.abs(v[~np.isnan(v)])
                    s = scale_for(mags.max() if mags.size else 0.0, self.form)
                    c = self.codes[side, slot, h]
                    if b * BLOCK < position:
                        was = self.scales[side, slot, h, b]
                        s = max(s, was)
                        if s != was:
                            old = slice(b * BLOCK, position)
                            c[old] = nearest(c[old] * (was / s), self.form)
                    c[new] = nearest(v / s, self.form)
                    self.scales[side, slot, h, b] = s
                    self.weights[slot, h, new] = 0.0

    def values(self, side, slot, h, rows):
        """The first `rows` rows of a head."""
        blocks = np.repeat(self.scales[side, slot, h], BLOCK)[:rows]
        return self.codes[side, slot, h, :rows] * blocks[:, None]

    def attend(self, slot, seen, q, scale):
        """One token's query heads [heads, head_dim] over the first `seen` rows: outputs, weights [heads, seen],
        and for each head the largest |q| |k| sum, and of |v| the weighted sum and the sum (for tolerances)."""
        kv = self.codes.shape[2]
        group = q.shape[0] // kv
        out, weights, size, mass = [], [], [], []
        for i in range(q.shape[0]):
            k, v = (self.values(side, slot, i // group, seen) for side in range(2))
            x = q[i].astype(np.float64)
            s = k @ x * scale
            if seen == 0:
                out.append(np.zeros(q.shape[1])), weights.append(s), size.append(0.0), mass.append(np.zeros((2, q.shape[1])))
                continue
            p = np.exp(s - s.max())
            p /= p.sum()
            out.append(p @ v), weights.append(p)
            size.append(float((np.abs(k) @ np.abs(x)).max() * scale)), mass.append(np.stack([p @ np.abs(v), np.abs(v).sum(0)]))
        return np.array(out), np.array(weights), np.array(size), np.array(mass)

    def keep(self, slot, h, rows, budget, first, last):
        """The rows of a head that an eviction keeps."""
        if rows <= budget:
            return list(range(rows))
        first = min(first, budget)
        last = min(last, budget - first)
        w = self.weights[slot, h].astype(np.float64)
        inner = sorted(range(first, rows - last), key=lambda r: (np.isnan(w[r]), -w[r] if not np.isnan(w[r]) else 0.0, r))
        return sorted(list(range(first)) + inner[:budget - first - last] + list(range(rows - last, rows)))

    def evict(self, slot, rows, budget, first, last, into=None, into_slot=None):
        """Returns the kept rows of each head, after moving them."""
        to = into or self
        to_slot = slot if into_slot is None else into_slot
        kept = []
        for h in range(self.codes.shape[2]):
            stay = self.keep(slot, h, rows, budget, first, last)
            kept.append(stay)
            for side in range(2):
                x = self.values(side, slot, h, rows)[stay]
                for b in range((len(stay) + BLOCK - 1) // BLOCK):
                    part = x[b * BLOCK:(b + 1) * BLOCK]
                    mags = np.abs(part[~np.isnan(part)])
                    s = scale_for(mags.max() if mags.size else 0.0, self.form)
                    to.codes[side, to_slot, h, b * BLOCK:b * BLOCK + len(part)] = nearest(part / s, self.form)
                    to.scales[side, to_slot, h, b] = s
            to.weights[to_slot, h, :len(stay)] = self.weights[slot, h, stay]
        return kept


def attend_bound(size, mass, rows, head_dim):
    """How far an output may be off. A score: queries as two fp16 halves (2^-22), sums of sixteen products cut off
    by the tensor core (2^-22 of them), head_dim / 16 fp32 additions and two products (2^-24 each): of the sum of
    |q| |k|. That twice (numerator and denominator), 2^-20 for exp2f, the halves of the weights and the products, and a
    2^-24 for each addition of the weighted rows (16 at a time, then warps and splits) and of their sum: of the weighted sum
    of |v|. The halves of a weight are fp16 numbers of it times 2^15, whose smallest step is 2^-24: a weight is 2^-40 off
    at the least, as a part of the largest one, so its row adds 2^-40 |v| however little it weighs."""
    score = size * (2.0 ** -22 + 2.0 ** -22 + (head_dim / 16 + 2) * 2.0 ** -24)
    weighted, whole = mass[..., 0, :], mass[..., 1, :]
    return (2 * score + 2.0 ** -20 + (rows / 16 + 64) * 2.0 ** -24)[..., None] * weighted + 2.0 ** -40 * whole


def frequencies(rope_dim, theta, scaling="none", factor=1.0, original=0.0, fast=32.0, slow=1.0):
    pairs = rope_dim // 2
    out = []
    low = high = 0
    if scaling == "by_parts":
        low, high = (rope_dim * math.log(original / (2 * math.pi * n)) / (2 * math.log(theta)) for n in (fast, slow))
        low, high = min(max(math.floor(low), 0), pairs - 1), min(max(math.ceil(high), 0), pairs - 1)
    for i in range(pairs):
        f = theta ** (-2.0 * i / rope_dim)
        if scaling == "linear":
            f /= factor
        elif scaling == "by_parts":
            part = min(1.0, max(0.0, (i - low) / max(high - low, 1e-3)))
            f = f * (1 - part) + f / factor * part
        out.append(f)
    return np.array(out)


def rope(x, positions, freq, layout, magnitude=1.0, norm=None, eps=0.0):
    """x: [tokens, heads, head_dim]. Returns the rotated rows, and the sum of magnitudes behind each value."""
    x = x.astype(np.float64)
    if norm is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * norm.astype(np.float64)
    pairs = len(freq)
    y, size = x.copy(), np.abs(x)
    # Whole turns go before the product is rounded: positions are split so that nothing is lost.
    turns = np.zeros((len(positions), pairs))
    for t, p in enumerate(positions):
        for i, f in enumerate(freq):
            turns[t, i] = math.fmod(float(p) * f, 2 * math.pi)
    c, s = np.cos(turns)[:, None, :] * magnitude, np.sin(turns)[:, None, :] * magnitude
    a, b = (slice(0, pairs), slice(pairs, 2 * pairs)) if layout == "halves" else (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2))
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    size[..., a] = size[..., b] = (np.abs(x[..., a]) + np.abs(x[..., b])) * abs(magnitude)
    return y, size
