"""Plain references of the paged-cache operators and of 4-bit weights: numpy in 64
bits, and page bookkeeping in Python loops."""
from __future__ import annotations

import numpy as np


def pages_for(n, page):
    return -(-n // page)


class Layout:
    """Sequences of the given lengths with their pages at random places of a pool;
    table entries past a sequence's pages are out of range on purpose."""

    def __init__(self, lens, page, seed, spare=2, columns=None):
        rng = np.random.default_rng(seed)
        need = [pages_for(n, page) for n in lens]
        self.lens, self.page = list(lens), page
        self.pages = sum(need) + spare
        self.columns = columns or max(need + [1]) + 1
        order = rng.permutation(self.pages)
        self.table = np.full((len(lens), self.columns), 2**30, dtype=np.int32)
        at = 0
        for b, k in enumerate(need):
            self.table[b, :k] = order[at:at + k]
            at += k

    def rows(self, b, n=None):
        """Pool rows of the first n cached rows of sequence b."""
        t = np.arange(self.lens[b] if n is None else n)
        return self.table[b, t // self.page].astype(np.int64) * self.page + t % self.page


def decode(q, k, v, scale):
    """One sequence and KV head in 64 bits: q [G, D], k, v [n, D] -> (out [G, D], bound
    [G, D]).  The bound is what fp16 outputs of kernels with fp32 sums and fp16 weights may
    be off: a weight's relative error e is half a step of fp16 (2^-11), the error of its
    score (D + 2 roundings of fp32 over the terms' magnitudes) and a few roundings of the
    exponential; weights below 2^-28 of the largest may lose 2^-39 of it; numerator and
    denominator are each off by e; sums of n terms add n / 16 + 64 roundings of fp32."""
    q, k, v = (np.asarray(x, dtype=np.float64) for x in (q, k, v))
    s = q @ k.T * scale
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    out = p @ v
    size = p @ np.abs(v)
    n, D = k.shape
    terms = (np.abs(q) @ np.abs(k).T).max(-1, keepdims=True) * scale
    e = 2.0**-11 + (D + 2) * 2.0**-24 * terms + 2.0**-20 + (n / 16 + 64) * 2.0**-24
    bound = 2 * e * size + 2.0**-11 * np.abs(out) + n * 2.0**-38 * np.abs(v).max() + 2.0**-24
    return out, bound


# ---------------------------------------------------------------- pages

class Pool:
    """Page bookkeeping, one page at a time."""

    def __init__(self, pages, page, max_pages, seqs, contents):
        self.page, self.max_pages = page, max_pages
        self.refs = [0] * pages
        self.table = [[-1] * max_pages for _ in range(seqs)]
        self.lens = [0] * seqs
        self.contents = contents  # [planes, pages, elements]

    def grow(self, amounts):
        """(missing pages, rows that are too short)"""
        need, copies, short = [], [], 0
        for b, g in enumerate(amounts):
            n = self.lens[b]
            need.append(0)
            copies.append(False)
            if g <= 0:
                continue
            if n + g > self.max_pages * self.page:
                short += 1
                continue
            copies[b] = n % self.page != 0 and self.refs[self.table[b][n // self.page]] > 1
            need[b] = pages_for(n + g, self.page) - pages_for(n, self.page) + copies[b]
        if short:
            return 0, short
        free = [p for p, r in enumerate(self.refs) if r == 0]
        if sum(need) > len(free):
            return sum(need) - len(free), 0
        free = iter(free)
        for b, g in enumerate(amounts):
            if g <= 0:
                continue
            n = self.lens[b]
            if copies[b]:
                old, new = self.table[b][n // self.page], next(free)
                self.contents[:, new] = self.contents[:, old]
                self.refs[old] -= 1
                self.refs[new] = 1
                self.table[b][n // self.page] = new
            for j in range(pages_for(n, self.page), pages_for(n + g, self.page)):
                self.table[b][j] = next(free)
                self.refs[self.table[b][j]] = 1
            self.lens[b] = n + g
        return 0, 0

    def free(self, keep=None):
        for b, n in enumerate(self.lens):
            k = 0 if keep is None else keep[b]
            if 0 <= k < n:
                for j in range(pages_for(k, self.page), pages_for(n, self.page)):
                    self.refs[self.table[b][j]] -= 1
                self.lens[b] = k

    def fork(self, parents):
        held = list(self.lens)
        for i, p in enumerate(parents):
            if not 0 <= p < len(held) or held[i] or p == i or parents[p] >= 0:
                continue
            for j in range(pages_for(held[p], self.page)):
                self.table[i][j] = self.table[p][j]
                self.refs[self.table[p][j]] += 1
            self.lens[i] = held[p]

    def compact(self):
        used = sum(r > 0 for r in self.refs)
        moves = dict(zip([p for p, r in enumerate(self.refs) if r and p >= used],
                         [p for p, r in enumerate(self.refs) if not r and p < used]))
        for a, b in moves.items():
            self.contents[:, b] = self.contents[:, a]
            self.refs[b], self.refs[a] = self.refs[a], 0
        for b, n in enumerate(self.lens):
            for j in range(pages_for(n, self.page)):
                self.table[b][j] = moves.get(self.table[b][j], self.table[b][j])
        return used


# ---------------------------------------------------------------- 4-bit weights

def w4_quantize(w, group):
    """(codes [N, K], scales fp16 [groups, N]) of fp16 weights."""
    N, K = w.shape
    groups = -(-K // group)
    scales = np.zeros((groups, N), dtype=np.float16)
    codes = np.full((N, K), 8, dtype=np.int64)
    x = w.astype(np.float32)
    for g in range(groups):
        part = x[:, g * group:(g + 1) * group]
        s = (np.abs(part).max(1) / np.float32(7)).astype(np.float16)
        scales[g] = s
        ok = s > 0
        with np.errstate(all="ignore"):
            c = np.rint(part / s.astype(np.float32)[:, None])
        c = np.clip(np.nan_to_num(c), -8, 7).astype(np.int64) + 8
        codes[ok, g * group:(g + 1) * group] = c[ok]
    return codes, scales


def w4_words(codes):
    """Codes [N, K] in the packed tile order, uint32."""
    N, K = codes.shape
    rt, ct = -(-N // 16), -(-K // 128)
    full = np.full((rt * 16, ct * 128), 8, dtype=np.uint64)
    full[:N, :K] = codes
    out = np.zeros((rt, ct, 4, 16, 4), dtype=np.uint64)
    for a in range(4):
        for s in range(4):
            for e in range(8):
                bits = 4 * (e // 2) + 16 * (e % 2)
                columns = full[:, 32 * s + 8 * a + e::128].reshape(rt, 16, ct)
                out[:, :, a, :, s] |= columns.transpose(0, 2, 1) << np.uint64(bits)
    return out.astype(np.uint32)


def w4_product(codes, scales, group, x, residual=None):
    """(y, bound): products in 64 bits; fp16 outputs with fp32 sums may be off by K + 16
    roundings of fp32 over the terms' magnitudes and half a step of fp16."""
    K = codes.shape[1]
    s = np.repeat(scales.astype(np.float64), group, axis=0)[:K].T
    w = (codes - 8) * s
    x = x.astype(np.float64)
    y, size = x @ w.T, np.abs(x) @ np.abs(w).T
    if residual is not None:
        y, size = y + residual.astype(np.float64), size + np.abs(residual.astype(np.float64))
    return y, (K + 16) * 2.0**-24 * size + 2.0**-11 * np.abs(y) + 2.0**-24
