"""Inputs, the 64-bit reference and the error bound for tree attention over the paged cache."""
from __future__ import annotations

import math

import numpy as np


class TreeCase:
    """Requests with committed and drafted tokens in paged fp16 pools; every pool row that belongs to no token is NaN."""

    def __init__(self, seed, prefix, draft, H, KVH, D, P=64, mask="tree", slack=3, fill=np.nan):
        rng = np.random.default_rng(seed)
        self.prefix, self.draft = np.array(prefix, np.uint32), np.array(draft, np.uint32)
        self.N, self.H, self.KVH, self.D, self.P = len(prefix), H, KVH, D, P
        need = [-(-(int(c) + int(d)) // P) for c, d in zip(prefix, draft)]
        self.capacity = sum(need) + slack
        self.pt_flat = rng.permutation(self.capacity)[: sum(need)].astype(np.uint32)
        self.pt_off = np.concatenate([[0], np.cumsum(need)]).astype(np.uint32)
        self.k = np.full((self.capacity, P, KVH, D), fill, np.float16)
        self.v = np.full((self.capacity, P, KVH, D), fill, np.float16)
        for r in range(self.N):
            for pos in range(int(prefix[r]) + int(draft[r])):
                page, slot = self.where(r, pos)
                self.k[page, slot] = rng.standard_normal((KVH, D)).astype(np.float16)
                self.v[page, slot] = rng.standard_normal((KVH, D)).astype(np.float16)
        self.T = int(self.draft.sum())
        self.q = rng.standard_normal((self.T, H, D)).astype(np.float32)
        self.sees = []
        for d in draft:
            see = np.zeros((d, d), bool)
            for i in range(d):
                if mask == "bits":
                    see[i] = rng.random(d) < 0.4
                elif mask == "tree":
                    parent = int(rng.integers(max(-1, i - 5), i))
                    if parent >= 0:
                        see[i] = see[parent]
                    see[i, i] = True
                elif mask == "chain":
                    see[i, : i + 1] = True
            self.sees.append(see)   # mask == "none": nobody sees a drafted token
        self.words = max(1, (max(draft, default=0) + 31) // 32)

    def where(self, r, pos):
        return int(self.pt_flat[self.pt_off[r] + pos // self.P]), pos % self.P

    @property
    def mask(self):
        rows = []
        for d, see in zip(self.draft, self.sees):
            wide = np.zeros((int(d), self.words * 32), bool)
            wide[:, : int(d)] = see
            rows.append(np.packbits(wide, axis=1, bitorder="little").view(np.uint32).reshape(int(d), self.words))
        return np.ascontiguousarray(np.concatenate(rows)) if rows else np.zeros((0, self.words), np.uint32)

    def tables(self):
        return self.pt_flat, self.pt_off, self.prefix, self.draft, self.mask


def reference(case, q, scale, exact_f32):
    """(O, bound) in 64 bits. Only tokens that a row sees are touched. The bound follows the kernels' arithmetic:

    - a score is an fp32 sum of D products, in whatever order and with truncation: D * 2^-23 * scale * sum |q k| at most,
      plus the rounding of the exponent's argument, 2^-22 of the largest score; fp32 queries enter as two fp16 halves,
      2^-22 of |q| (each weight is off by that much, relatively, twice: it enters numerator and denominator)
    - a weight is rounded to fp16 before it meets V: 2^-11 (2^-22 when it is carried in two halves), and at least the
      subnormal step, 2^-25 of a weight of 1, where the largest weight is at least 1
    - the sum over S tokens is fp32: S * 2^-23 of the sum of magnitudes at most, and the exponential 2^-21
    - the result is rounded once: 2^-11 of the value for fp16, 2^-24 for fp32
    """
    H, KVH, D = case.H, case.KVH, case.D
    out = np.zeros((case.T, H, D))
    tol = np.zeros((case.T, H, D))
    t = 0
    for r in range(case.N):
        c, d = int(case.prefix[r]), int(case.draft[r])
        places = [case.where(r, p) for p in range(c + d)]
        for i in range(d):
            seen = list(range(c)) + [c + j for j in np.flatnonzero(case.sees[r][i])]
            if seen:
                k = np.stack([case.k[places[p]] for p in seen]).astype(np.float64)   # [S, KVH, D]
                v = np.stack([case.v[places[p]] for p in seen]).astype(np.float64)
                for h in range(H):
                    kh, vh = k[:, h // (H // KVH)], v[:, h // (H // KVH)]
                    qh = q[t + i, h].astype(np.float64)
                    s = scale * (kh @ qh)
                    size = scale * (np.abs(kh) @ np.abs(qh))
                    w = np.exp(s - s.max())
                    total = w.sum()
                    o = (w @ vh) / total
                    mag = (w @ np.abs(vh)) / total
                    e = (D * 2.0**-23 + 2.0**-22) * size.max() + 2.0**-22 * np.abs(s).max()
                    weight = 2.0**-22 if exact_f32 else 2.0**-11
                    out[t + i, h] = o
                    tol[t + i, h] = ((2 * e + weight + len(seen) * 2.0**-23 + 2.0**-21) * mag
                                     + len(seen) * 2.0**-25 * np.abs(vh).max() / total
                                     + (2.0**-24 if exact_f32 else 2.0**-11) * np.abs(o) + 1e-30)
        t += d
    return out, tol


def default_scale(case):
    return 1.0 / math.sqrt(case.D)
