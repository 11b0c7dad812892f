"""The operators of a decoding step in plain 64-bit Python, one element after another: what the GPU tests compare with."""
import math

import numpy as np
import torch

TORCH = {"bf16": torch.bfloat16, "f16": torch.float16}


def step(dtype):
    """Half a step of the type, relative to the value."""
    return torch.finfo(TORCH[dtype]).eps / 2


def smallest(dtype):
    """Half the distance between the type's smallest numbers."""
    return float(torch.finfo(TORCH[dtype]).smallest_normal) * torch.finfo(TORCH[dtype]).eps / 2


# ------------------------------------------------------------------------------------------------ pages
class Pool:
    def __init__(self, sequences, width, pages, page_size):
        self.table = [[-1] * width for _ in range(sequences)]
        self.length, self.held, self.refcount = [0] * sequences, [0] * sequences, [0] * pages
        self.width, self.page_size = width, page_size

    def _free(self):
        return [p for p, c in enumerate(self.refcount) if c == 0]

    def reserve(self, extra):
        want = [-(-(n + e) // self.page_size) if e >= 0 else 0 for n, e in zip(self.length, extra)]
        if any(w > self.width for w in want):
            return 2
        free = self._free()
        if sum(max(0, w - h) for w, h in zip(want, self.held)) > len(free):
            return 1
        for s, w in enumerate(want):
            while self.held[s] < w:
                page = free.pop(0)
                self.table[s][self.held[s]] = page
                self.refcount[page] = 1
                self.held[s] += 1
        return 0

    def free(self, which):
        for s, w in enumerate(which):
            if w:
                for j in range(self.held[s]):
                    self.refcount[self.table[s][j]] -= 1
                    self.table[s][j] = -1
                self.length[s] = self.held[s] = 0

    def fork(self, parent):
        """Returns (status, [(source page, new page, filled slots)])."""
        n, ps = len(self.table), self.page_size
        child = [0 <= p < n and p != s for s, p in enumerate(parent)]
        before = [list(r) for r in self.table]
        length, held, free, copies = list(self.length), list(self.held), self._free(), []
        if sum(c and length[p] % ps != 0 for c, p in zip(child, parent)) > len(free):
            return 1, []
        for s, p in enumerate(parent):
            if not child[s]:
                continue
            full = length[p] // ps
            row = before[p][:full] + [-1] * (self.width - full)
            for page in row[:full]:
                self.refcount[page] += 1
            if length[p] % ps:
                row[full] = free.pop(0)
                self.refcount[row[full]] += 1
                copies.append((before[p][full], row[full], length[p] % ps))
            for page in before[s][:held[s]]:
                self.refcount[page] -= 1
            self.table[s], self.length[s], self.held[s] = row, length[p], -(-length[p] // ps)
        return 0, copies

    def place(self, s, pos):
        """(page, slot) or None."""
        j = pos // self.page_size
        if pos < 0 or j >= min(self.held[s], self.width) or not 0 <= self.table[s][j] < len(self.refcount):
            return None
        return self.table[s][j], pos % self.page_size

    def path(self, s, path):
        """The moves of an accepted path: [(from, to)] as (page, slot)."""
        moves, before = [], -1
        for i, node in enumerate(path):
            a, b = self.place(s, self.length[s] + node), self.place(s, self.length[s] + i)
            if node <= before or a is None or b is None:
                break
            moves.append((a, b))
            before = node
        return moves


# ------------------------------------------------------------------------------------------------ rotary positions
def frequencies(rotary, base, kind="none", factor=1.0, span=0.0, low=0.0, high=0.0):
    f = [base ** (-2.0 * i / rotary) for i in range(rotary // 2)]
    if kind == "linear":
        return [x / factor for x in f], 1.0
    if kind == "stretched":
        b = base * factor ** (rotary / (rotary - 2)) if rotary > 2 else base
        return [b ** (-2.0 * i / rotary) for i in range(rotary // 2)], 1.0
    if kind == "yarn":
        pair = lambda turns: rotary / 2 * math.log(span / (turns * 2 * math.pi), base)  # noqa: E731
        a, z = max(math.floor(pair(high)), 0), min(math.ceil(pair(low)), rotary - 1)
        mix = [min(1.0, max(0.0, (i - a) / max(z - a, 0.001))) for i in range(len(f))]
        return [x / factor * w + x * (1 - w) for x, w in zip(f, mix)], 0.1 * math.log(factor) + 1
    if kind == "banded":
        mix = [min(1.0, max(0.0, (span * x / (2 * math.pi) - low) / (high - low))) for x in f]
        return [x * ((1 - w) / factor + w) for x, w in zip(f, mix)], 1.0
    return f, 1.0


def rotate(x, positions, f, magnitude, interleaved):
    """x [rows][heads][dim] float64; also the largest factor of an element's error in a cosine or sine."""
    y, size = x.copy(), np.zeros_like(x)
    half = len(f)
    for i, w in enumerate(f):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = np.cos(np.asarray(positions, np.float64) * w)[:, None], np.sin(np.asarray(positions, np.float64) * w)[:, None]
        y[..., a], y[..., b] = magnitude * (x[..., a] * c - x[..., b] * s), magnitude * (x[..., b] * c + x[..., a] * s)
        size[..., a] = size[..., b] = magnitude * (np.abs(x[..., a]) + np.abs(x[..., b]))
    return y, size


# ------------------------------------------------------------------------------------------------ attention
def attention(q, pool, k, v, row_start, mask_bits, scale, dtype):
    """q [rows][heads][dim] float64; k, v [pages][slots][cache heads][dim] float64; mask_bits [rows][nodes] bool or None (a chain).
    Returns (out, bound), NaN where no row of a sequence stands."""
    rows, hq, dim = q.shape
    out, bound = np.full(q.shape, np.nan), np.zeros(q.shape)
    per = hq // k.shape[2]
    for s in range(len(pool.table)):
        for r in range(max(row_start[s], 0), min(row_start[s + 1], rows)):
            node, nodes = r - row_start[s], min(row_start[s + 1], rows) - row_start[s]
            seen = list(range(pool.length[s]))
            for m in range(nodes):
                if (m <= node) if mask_bits is None else (m < mask_bits.shape[1] and mask_bits[r, m]):
                    seen.append(pool.length[s] + m)
            at = [pool.place(s, p) for p in seen]
            at = [x for x in at if x is not None]
            for h in range(hq):
                if not at:
                    out[r, h] = 0
                    continue
                ks = np.array([k[p, t, h // per] for p, t in at])
                vs = np.array([v[p, t, h // per] for p, t in at])
                with np.errstate(invalid="ignore", over="ignore"):
                    sc = scale * (ks @ q[r, h])
                    w = np.exp(sc - sc.max())
                    w /= w.sum()
                    out[r, h] = (w[:, None] * vs).sum(0)
                    size = (w[:, None] * np.abs(vs)).sum(0)
                    # a weight is off by the error of its score (dim products in fp32, the product with the scale, the difference from
                    # the maximum), the exponential's 2^-22 and its rounding; the sums by a 2^-23 of their size for every term that the
                    # tensor cores cut off; the total likewise; the result by its rounding
                    score = (dim + 8) * 2.0**-24 * scale * (np.abs(ks) @ np.abs(q[r, h])).max()
                    bound[r, h] = (step(dtype) + 2 * score + (2 * len(at) + 64) * 2.0**-23) * size + step(dtype) * np.abs(out[r, h]) + \
                        smallest(dtype) * (1 + np.abs(vs).sum(0) / max(np.exp(sc - sc.max()).sum(), 1))
    return out, bound
