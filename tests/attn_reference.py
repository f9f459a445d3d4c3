"""Attention and the 8-bit key / value cache in 64 bits, and the error bounds that the kernels are held to.

Bounds.  u = half a step of the output's type (bf16 2^-8, f16 2^-11, f32 2^-24).  With o = sum_j p_j v_j and A = sum_j p_j |v_j|:
  rounding the result                       u |o|
  probabilities rounded to a type of half step u_p before the second product: each p_j is off by u_p p_j       u_p A
  scores: f32 sums of hd products, off by at most (hd + 2) 2^-24 sum |q k| scale <= E, and the argument of the exponential is rounded
  once more, so every p_j is off by a factor of e^(2 E') - 1, E' = E + 2^-20; sums over j in f32 in 64 or more partial sums: below 2^-19 A
"""
import numpy as np

HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def attend(q, k, v, last, scale):
    """q [rows][hd], k / v [len][hd] f64; row r sees 0 .. last[r].  Returns (o, A, E) with E the largest sum |q k| scale of a row."""
    o, a, e = np.zeros((q.shape[0], v.shape[1])), np.zeros((q.shape[0], v.shape[1])), np.zeros(q.shape[0])
    for r in range(q.shape[0]):
        n = int(last[r]) + 1
        if n <= 0:
            continue
        s = k[:n] @ q[r] * scale
        p = np.exp(s - s.max())
        p /= p.sum()
        o[r], a[r] = p @ v[:n], p @ np.abs(v[:n])
        e[r] = (np.abs(k[:n]) @ np.abs(q[r])).max() * scale
    return o, a, e


def tolerance(o, a, e, hd, u, u_p):
    score = (hd + 2) * 2.0 ** -24 * e + 2.0 ** -20
    return u * np.abs(o) * 1.01 + (u_p + np.expm1(2 * score)[:, None] + 2.0 ** -19) * a + 1e-30


def pow2_scale(amax, limit):
    """The smallest power of two, at least 2^-100, with amax <= limit * scale; at most the one whose multiples stay below 2^128."""
    e, most = -100, 128 - int(np.ceil(np.log2(limit)))
    while amax > limit * 2.0 ** e and e < most:
        e += 1
    return 2.0 ** e


_E4M3 = np.array(sorted({m * 2.0 ** -9 for m in range(8)} | {(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)
                                                             if not (e == 15 and m == 7)}))


def round_e4m3(x):
    """To the nearest of e4m3's values, ties to the even mantissa."""
    a = np.abs(x)
    i = np.clip(np.searchsorted(_E4M3, a), 1, len(_E4M3) - 1)
    lo, hi = _E4M3[i - 1], _E4M3[i]
    up = (a - lo > hi - a) | ((a - lo == hi - a) & (i % 2 == 0))         # the value's index has the parity of its mantissa
    return np.sign(x) * np.where(up, hi, lo)


LIMIT = {"s8": 127.0, "e4m3": 448.0}


def round8(x, fmt):
    x = np.clip(x, -LIMIT[fmt], LIMIT[fmt])
    return np.rint(x) if fmt == "s8" else round_e4m3(x)


class Model:
    """The cache and its page operations, in Python lists and f64 values."""

    def __init__(self, n_pages, max_seqs, max_pages, page, kv_heads, hd, fmt, layers=1):
        self.n_pages, self.max_seqs, self.max_pages, self.page, self.fmt, self.layers = n_pages, max_seqs, max_pages, page, fmt, layers
        self.refs, self.lens, self.tail = [0] * n_pages, [0] * max_seqs, [0] * max_seqs
        self.table = [[-1] * max_pages for _ in range(max_seqs)]
        self.q = {t: np.zeros((layers, n_pages, kv_heads, page, hd)) for t in "kv"}
        self.scale = {t: np.zeros((layers, n_pages, kv_heads)) for t in "kv"}
        self.result = [0, 0, 0, 0]

    def pages(self, n):
        return -(-n // self.page)

    def free(self):
        return [p for p in range(self.n_pages) if self.refs[p] == 0]

    def _refuse(self, status, needed=0):
        self.result = [status, len(self.free()), 0, needed]

    def _bad(self, ids):
        return any(not 0 <= i < self.max_seqs for i in ids) or len(set(ids)) < len(ids)

    def extend(self, seqs, add):
        if self._bad(seqs) or any(n < 0 or self.lens[s] + n > self.max_pages * self.page for s, n in zip(seqs, add)):
            for s in seqs:
                if 0 <= s < self.max_seqs:
                    self.tail[s] = 0
            return self._refuse(-1)
        need = [self.pages(self.lens[s] + n) - self.pages(self.lens[s]) for s, n in zip(seqs, add)]
        free = self.free()
        if sum(need) > len(free):
            for s in seqs:
                self.tail[s] = 0
            return self._refuse(-3, sum(need))
        for s, n in zip(seqs, add):
            for p in range(self.pages(self.lens[s]), self.pages(self.lens[s] + n)):
                self.table[s][p] = free.pop(0)
                self.refs[self.table[s][p]] = 1
            self.lens[s] += n
            self.tail[s] = n
        self.result = [0, len(free), sum(need), sum(need)]

    def _copy(self, pairs):
        for src, dst in pairs:
            for t in "kv":
                self.q[t][:, dst], self.scale[t][:, dst] = self.q[t][:, src], self.scale[t][:, src]

    def truncate(self, seqs, lens=None):
        lens = [0] * len(seqs) if lens is None else lens
        if self._bad(seqs) or any(not 0 <= n <= self.lens[s] for s, n in zip(seqs, lens)):
            return self._refuse(-1)
        refs = list(self.refs)
        for s, n in zip(seqs, lens):
            for p in self.table[s][self.pages(n):self.pages(self.lens[s])]:
                refs[p] -= 1
        cut = [i for i, (s, n) in enumerate(zip(seqs, lens)) if n % self.page and refs[self.table[s][n // self.page]] > 1]
        free = [p for p in range(self.n_pages) if refs[p] == 0]
        if len(cut) > len(free):
            return self._refuse(-3, len(cut))
        self.refs = refs
        for s, n in zip(seqs, lens):
            for p in range(self.pages(n), self.pages(self.lens[s])):
                self.table[s][p] = -1
            self.lens[s], self.tail[s] = n, 0
        pairs = []
        for i in cut:
            s, at = seqs[i], lens[i] // self.page
            pairs.append((self.table[s][at], free.pop(0)))
            self.refs[pairs[-1][0]] -= 1
            self.refs[pairs[-1][1]] = 1
            self.table[s][at] = pairs[-1][1]
        self._copy(pairs)
        self.result = [0, len(self.free()), len(cut), len(cut)]

    def fork(self, src, dst, share):
        if self._bad(dst) or any(not 0 <= s < self.max_seqs for s in src) or set(src) & set(dst) or any(self.lens[d] for d in dst):
            return self._refuse(-1)
        first = [self.lens[s] // self.page if share else 0 for s in src]
        need = sum(self.pages(self.lens[s]) - f for s, f in zip(src, first))
        free = self.free()
        if need > len(free):
            return self._refuse(-3, need)
        pairs = []
        for s, d, f in zip(src, dst, first):
            for p in range(self.pages(self.lens[s])):
                page = self.table[s][p]
                if p < f:
                    self.refs[page] += 1
                else:
                    pairs.append((page, free.pop(0)))
                    page = pairs[-1][1]
                    self.refs[page] = 1
                self.table[d][p] = page
            self.lens[d], self.tail[d] = self.lens[s], 0
        self._copy(pairs)
        self.result = [0, len(free), need, need]

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        high = [p for p in range(live, self.n_pages) if self.refs[p] > 0]
        pairs = list(zip(high, [p for p in range(live) if self.refs[p] == 0]))
        self._copy(pairs)
        to = dict(pairs)
        for a, b in pairs:
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        self.result = [0, self.n_pages - live, len(pairs), len(pairs)]

    def append(self, layer, name, s, x):
        """x [n][kv_heads][hd] f64: the tokens of sequence s's last extension."""
        n, page = x.shape[0], self.page
        first = self.lens[s] - n
        q, scale = self.q[name][layer], self.scale[name][layer]
        for p in range(first // page, self.pages(self.lens[s])):
            a, b = max(first, p * page), min(self.lens[s], (p + 1) * page)
            if a >= b:
                continue
            pid, held = self.table[s][p], a - p * page
            for h in range(x.shape[1]):
                new = x[a - first:b - first, h]
                old = scale[pid, h] if held else 0.0
                if not np.isfinite(new).all() or not np.isfinite(old):
                    scale[pid, h] = np.nan
                    q[pid, h, held:b - p * page] = 0.0
                    continue
                sc = max(old, pow2_scale(np.abs(new).max(), LIMIT[self.fmt]))
                if held:
                    q[pid, h, :held] = round8(q[pid, h, :held] * (old / sc), self.fmt)
                q[pid, h, held:b - p * page] = round8(new / sc, self.fmt)
                scale[pid, h] = sc

    def read(self, layer, name, s):
        """[len][kv_heads][hd]"""
        pids = self.table[s][:self.pages(self.lens[s])]
        x = self.q[name][layer][pids] * self.scale[name][layer][pids][..., None, None]
        return x.transpose(0, 2, 1, 3).reshape(-1, x.shape[1], x.shape[3])[:self.lens[s]] if pids else np.zeros((0,) + self.q[name].shape[2:5:2])
