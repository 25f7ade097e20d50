"""Tree speculation in 64 bits, as its rules are written, for the tests."""
from __future__ import annotations

import numpy as np

import oracle as O

ROW_BYTES = {1: 34, 2: 18}   # of 32 values, by kv_dtype


def chain(n):
    return [-1] + list(range(n - 1))


def star(n):
    return [-1] + [0] * (n - 1)


def random_tree(rng, n, width=4):
    return [-1] + [int(rng.integers(max(0, i - width), i)) for i in range(1, n)]


def sees(parents, node):
    """The drafted rows that a node sees."""
    got = []
    while node >= 0:
        got.append(node)
        up = parents[node]
        node = up if -1 <= up < node else -1
    return got


class Caches:
    """K and V of several slots in one cache format, with the values that they stand for.

    Rows that are not set hold `fill` (bytes), so that a read of them shows."""

    def __init__(self, kv_dtype, slots, kv, dim, stride, fill=0xFF, pad=0):
        self.kv_dtype, self.slots, self.kv, self.dim, self.stride = kv_dtype, slots, kv, dim, stride
        self.row = dim * 4 if kv_dtype == 0 else dim // 32 * ROW_BYTES[kv_dtype]
        self.slot_bytes = kv * stride * self.row + pad
        self.bytes = [np.full(slots * self.slot_bytes, fill, dtype=np.uint8) for _ in range(2)]
        self.values = [np.full((slots, kv, stride, dim), np.nan) for _ in range(2)]

    def rows(self, which, slot):
        """A view of a slot's rows: [kv][stride][row bytes], whatever the layout."""
        b = self.bytes[which][slot * self.slot_bytes:][:self.kv * self.stride * self.row]
        if self.kv_dtype == 0:
            return b.reshape(self.stride, self.kv, self.row).transpose(1, 0, 2)
        return b.reshape(self.kv, self.stride, self.row)

    def put(self, which, slot, row, x):
        """Rows [row, row + n) of a slot: x f32 [kv][n][dim]."""
        n = x.shape[1]
        x = np.ascontiguousarray(x, dtype=np.float32)
        if self.kv_dtype == 0:
            raw, back = x.view(np.uint8).reshape(self.kv, n, self.row), x
        else:
            enc, dec = ((O.quantize_q8, O.dequantize_q8), (O.quantize_q4, O.dequantize_q4))[self.kv_dtype - 1]
            raw = enc(x)
            back = dec(raw).reshape(x.shape)
            raw = raw.reshape(self.kv, n, self.row)
        self.rows(which, slot)[:, row:row + n] = raw
        self.values[which][slot, :, row:row + n] = back

    def fill(self, rng, slot, rows, k_scale=1.0, v_scale=1.0):
        for which, scale in ((0, k_scale), (1, v_scale)):
            self.put(which, slot, 0, scale * rng.standard_normal((self.kv, rows, self.dim)))


def attention(caches, slot, base, live, parents, q, heads, scale):
    """(out, bound): [live][heads][dim] in 64 bits, and how far 32-bit arithmetic over operands of 22 bits may be off.

    With u = 2^-23 (a sum in 32 bits that may be cut off, not rounded) and operands split into two 11-bit parts, each of
    which is rounded (2^-22 of the value, and the product of the two remainders 2^-22): a score's error is at most
    (2^-22 + 2 * 2^-22 + (3 * 16 + 8) u) * scale * sum |q k|, for 16 steps of three products each; one of 2^-22 of the score
    comes from the exponential's argument. Weights are off by that and by 2^-21 (the exponential); the sums over n rows by
    (3 n / 16 + 64) u of the sum of the weights times |v|, and the folds of the runs by another 64 u.

    Weights are not exact to 2^-22 of themselves however small they are. Their last bit is f16's 2^-24, they are kept 2^10
    times 2^(s + E - m), and m is at most the largest s + E and one half; so row j's weight is off by 2^-25 - 10 + 1/2 of
    2^(max (s + E)), its values, below 2^(E_j + 11) each, are multiplied back by 2^-E_j, and a tile's E is at most 7 above
    that of any of its rows, whose largest value is 2^(E + 10) or more: altogether less than 2^-35 + 1/2 + 7 + 1 of the largest
    p_j max |v_j| per row, n 2^-26 of it."""
    kv, dim = caches.kv, caches.dim
    group = heads // kv
    out, bound = np.zeros((live, heads, dim)), np.zeros((live, heads, dim))
    u, split = 2.0 ** -23, 2.0 ** -22
    for i in range(live):
        rows = np.array(list(range(base)) + sorted(base + j for j in sees(parents, i)), dtype=int)
        for h in range(heads):
            k, v = (caches.values[w][slot, h // group][rows] for w in range(2))
            x = q[i, h].astype(np.float64)
            s = scale * (k @ x)
            off = (3 * split + (3 * 16 + 8) * u) * scale * (np.abs(k) @ np.abs(x)) + split * np.abs(s)
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h] = p @ v
            most = off.max()   # (of a weight and of the whole: twice)
            bound[i, h] = (2 * most + 2.0 ** -20 + (3 * len(rows) / 16 + 128) * u) * (p @ np.abs(v))
            bound[i, h] += len(rows) * 2.0 ** -26 * (p * np.abs(v).max(1)).max()
    return out, bound


def probability(x):
    """What is no probability counts as 0."""
    x = np.asarray(x, dtype=np.float64)
    return np.where((x > 0) & np.isfinite(x), x, 0.0)


def verify(parents, tokens, target, draft, u, live):
    """(path, next) of a slot: target [nodes][vocab], draft the same or None, u [nodes]."""
    u = np.asarray(u, dtype=np.float64)
    vocab = target.shape[1]
    here, path = 0, [0]
    while True:
        r, found = probability(target[here]), -1
        for c in range(here + 1, live):
            x = int(tokens[c])
            if parents[c] != here or not 0 <= x < vocab:
                continue
            q = probability(draft[here]) if draft is not None else np.eye(1, vocab, x)[0]
            if u[c] * q[x] < r[x]:
                found = c
                break
            rest = np.maximum(r - q, 0.0)
            if rest.sum() > 0:
                r = rest / rest.sum()
        if found < 0:
            break
        here = found
        path.append(here)
    if not (r > 0).any():
        return path, -1
    run = np.cumsum(r)
    past = np.flatnonzero((run > u[0] * run[-1]) & (r > 0))
    return path, int(past[0]) if len(past) else int(np.flatnonzero(r > 0)[-1])
