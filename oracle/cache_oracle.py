"""CPU restatement of the attention cache's operators, for the tests only.

* ``rotary``: the pairs of the rotated channels as complex numbers times
  exp(i * position * freq), in float64.
* ``Pool``: pages, tables and holder counts as Python lists; reserve, free,
  fork, compact and copy one entry after the other.
* ``paged_attn``: softmax attention of one token per row over the visible keys
  of its sequence, in float64, with the bound that a 16-bit kernel's error obeys.
"""

from __future__ import annotations

import numpy as np


def rotary(x: np.ndarray, positions: np.ndarray, freqs: np.ndarray, offset: int, interleaved: bool,
           inverse: bool = False, amplitude: float = 1.0) -> np.ndarray:
    """x [..., H, D], positions [...] -> float64 [..., H, D]."""
    x = np.asarray(x, np.float64)
    half = len(freqs)
    angle = np.asarray(positions, np.float64)[..., None] * np.asarray(freqs, np.float64)
    w = np.exp((-1j if inverse else 1j) * angle)[..., None, :] * amplitude
    a = offset + (2 * np.arange(half) if interleaved else np.arange(half))
    b = a + (1 if interleaved else half)
    z = (x[..., a] + 1j * x[..., b]) * w
    y = x.copy()
    y[..., a], y[..., b] = z.real, z.imag
    return y


def rotary_bound(x: np.ndarray, y: np.ndarray, freqs: np.ndarray, offset: int, interleaved: bool, eps: float,
                 tiny: float, amplitude: float = 1.0) -> np.ndarray:
    """Largest error of a rotation in 32 bits, rounded once to a type of the given
    eps: half a step of the result (or half the least number ``tiny`` that is not
    zero), and before it, relative to |a| + |b|, 9.4e-8 from the angle (half a step
    of a fraction of a turn below 1/2: 2^-26 turns), one unit of 2^-24 each from the
    cosine, the amplitude, the product and the sum: 3.4e-7 together, 4e-7 here."""
    half = len(freqs)
    a = offset + (2 * np.arange(half) if interleaved else np.arange(half))
    b = a + (1 if interleaved else half)
    both = np.zeros(x.shape)
    both[..., a] = both[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
    calc = 4e-7 * amplitude * both
    moved = both > 0
    return np.where(moved, calc + eps / 2 * (np.abs(y) + calc) + tiny / 2, 0.0)


class Pool:
    """A cache's tables on lists: ``table`` [S][M], ``lens`` [S], ``refs`` [P]; ``pages``
    [L, P, page, D] any numpy array (or None)."""

    def __init__(self, table, lens, refs, page, pages=None):
        self.table, self.lens, self.refs = [list(r) for r in table], list(lens), list(refs)
        self.page, self.pages = page, pages
        self.bad = False      # an entry was refused
        self.short = False    # too few free pages

    def _pages(self, n):
        return -(-n // self.page)

    def reserve(self, seqs, lens):
        seen, plan = set(), []
        for s, n in zip(seqs, lens):
            if s < 0:
                continue
            ok = s < len(self.lens) and s not in seen and n >= 0 and self._pages(n) <= len(self.table[0])
            # the first entry that names a sequence claims it, whether or not its length fits
            seen.add(s)
            if not ok:
                self.bad = True
                continue
            plan.append((s, n))
        free = [p for p, r in enumerate(self.refs) if r <= 0]
        if sum(max(0, self._pages(n) - self._pages(self.lens[s])) for s, n in plan) > len(free):
            self.short = True
            return
        for s, n in plan:
            for j in range(self._pages(self.lens[s]), self._pages(n)):
                self.table[s][j] = free.pop(0)
                self.refs[self.table[s][j]] = 1
            self.lens[s] = max(self.lens[s], n)

    def free(self, seqs):
        for s in seqs:
            if s < 0:
                continue
            if s >= len(self.lens):
                self.bad = True
                continue
            for p in self.table[s]:
                if p >= 0:
                    self.refs[p] -= 1
            self.table[s] = [-1] * len(self.table[s])
            self.lens[s] = 0

    def fork(self, parents, children, lens=None):
        seen, plan, before = set(), [], list(self.lens)
        for i, (a, b) in enumerate(zip(parents, children)):
            if a < 0 or b < 0:
                continue
            ok = a < len(before) and b < len(before) and b not in seen and before[b] == 0
            seen.add(b)
            n = -1
            if ok:
                n = before[a] if lens is None else lens[i]
                ok = 0 <= n <= before[a]
            if not ok:
                self.bad = True
                continue
            plan.append((a, b, n))
        free = [p for p, r in enumerate(self.refs) if r <= 0]
        if sum(n % self.page != 0 for _, _, n in plan) > len(free):
            self.short = True
            return
        for a, b, n in plan:
            for j in range(n // self.page):
                self.table[b][j] = self.table[a][j]
                self.refs[self.table[a][j]] += 1
            if n % self.page:
                p, j = free.pop(0), n // self.page
                self.table[b][j], self.refs[p] = p, 1
                if self.pages is not None:
                    self.pages[:, p, :n % self.page] = self.pages[:, self.table[a][j], :n % self.page]
            self.lens[b] = n

    def compact(self):
        used = [p for p, r in enumerate(self.refs) if r > 0]
        n = len(used)
        holes = [p for p in range(n) if self.refs[p] <= 0]
        to = {p: p for p in used}
        for hole, p in zip(holes, [p for p in used if p >= n]):
            to[p] = hole
            self.refs[hole], self.refs[p] = self.refs[p], 0
            if self.pages is not None:
                self.pages[:, hole] = self.pages[:, p]
        self.table = [[to[p] if p >= 0 else -1 for p in row] for row in self.table]
        return [to.get(p, -1) for p in range(len(self.refs))]


def visible(position: int, window: int, first: int) -> np.ndarray:
    keys = np.arange(position + 1)
    return keys if not window else keys[(keys > position - window) | (keys < first)]


def paged_attn(q, kv_of, positions, sink, scale, window=0, first=0, half_step=0.0, tiny=0.0, weight_tiny=None):
    """q [T,H,D]; kv_of(t, keys) -> rows of row t's sequence; positions [T] (negative:
    padding).  Returns float64 out [T,H,D] and the largest error of a kernel that rounds
    the weights p and the output to a type with the given half step (relative):

    with weights p_j (1 + d_j), |d_j| <= half_step, summed as rounded, the quotient is off
    by at most half_step (sum p|kv| + |out|) to first order, its rounding by another
    half_step |out|; weights below the type's normal range are off by weight_tiny / 2 of the
    largest weight each (default: tiny, where the largest weight is at least 1 before the
    division; tiny / 2^k where it is at least 2^k).  That term grows with the number of
    keys: without a k it hides the loss of many small weights.  Scores and exponentials in 32
    bits add a relative 1e-4 at most (|z| < 100, 512 products: 512 2^-24 times
    scale sum |q k| < 30, and 2^-22 |z|), taken as 3e-4 of sum p|kv| + |out|."""
    q = np.asarray(q, np.float64)
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for t in range(q.shape[0]):
        if positions[t] < 0:
            continue
        keys = visible(int(positions[t]), window, first)
        kv = np.asarray(kv_of(t, keys), np.float64)
        if kv.shape[0] == 0:
            continue
        z = q[t] @ kv.T * scale                                          # [H, keys]
        s = np.full(q.shape[1], -np.inf) if sink is None else np.asarray(sink, np.float64)
        top = z.max(1)
        m = np.maximum(top, s)
        p = np.exp(z - m[:, None])
        den = p.sum(1) + np.exp(s - m)
        p /= den[:, None]
        out[t] = p @ kv
        spread = p @ np.abs(kv) + np.abs(out[t])
        largest = np.exp(top - m) / den
        small = (tiny if weight_tiny is None else weight_tiny) / 2 * largest[:, None] * np.abs(kv).sum(0)[None]
        bound[t] = (1.02 * half_step + 3e-4) * spread + half_step * np.abs(out[t]) + small + tiny / 2
    return out, bound
