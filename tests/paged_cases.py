"""Plain 64-bit implementations of the paged-cache operators and of draft verification, and the inputs
the tests run them on.  Everything here is torch or numpy on the CPU."""
from __future__ import annotations

import math

import numpy as np
import torch

D = 128
NAN_CODE = 0x7F


def code_values(codes: torch.Tensor) -> torch.Tensor:
    """e4m3 bytes as 64-bit values."""
    return codes.view(torch.uint8).view(torch.float8_e4m3fn).float().double()


def power_scale(amax: float) -> float:
    """The smallest power of two s with amax <= 448 s (at least 2^-64), 0 for 0."""
    if not amax > 0:
        return 0.0
    m, e = math.frexp(amax)
    return max(2.0 ** (e - 9 + (1 if m > 0.875 else 0)), 2.0 ** -64)


class Case:
    """Sequences (new tokens, length), their pages in a shuffled pool, and the pool itself on the CPU."""

    def __init__(self, seqs, page: int, kv_heads: int, seed: int, spare_pages: int = 3, level: float = 1.0):
        self.seqs, self.page, self.kv = seqs, page, kv_heads
        self.g = torch.Generator().manual_seed(seed)
        used = [-(-n // page) for _, n in seqs]
        self.pages = sum(used) + spare_pages
        perm = torch.randperm(self.pages, generator=self.g).to(torch.int32)
        self.table = torch.full((len(seqs), max(used + [1]) + 1), -1, dtype=torch.int32)
        for b, n in enumerate(used):
            self.table[b, :n] = perm[sum(used[:b]):sum(used[:b]) + n]
        self.cu = torch.tensor([0] + [sum(q for q, _ in seqs[:b + 1]) for b in range(len(seqs))], dtype=torch.int32)
        self.lens = torch.tensor([n for _, n in seqs], dtype=torch.int32)
        self.tokens = int(self.cu[-1])
        self.max_q, self.max_len = max(q for q, _ in seqs), max(n for _, n in seqs)
        # every code, scales of several sizes; a page's size differs by head
        shape = (self.pages, kv_heads, page, D)
        self.k, self.v = (self._codes(shape) for _ in range(2))
        self.ks, self.vs = (level * 2.0 ** torch.randint(-7, -3, shape[:2], generator=self.g).float() for _ in range(2))

    def _codes(self, shape):
        x = torch.randn(shape, generator=self.g) * 40
        return x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)

    def randn(self, *shape):
        return torch.randn(*shape, generator=self.g)

    def spoil_unused(self):
        """NaN codes and scales wherever no sequence has a position."""
        used = torch.zeros(self.pages, self.page, dtype=torch.bool)
        for b, (_, n) in enumerate(self.seqs):
            for j in range(n):
                used[self.table[b, j // self.page], j % self.page] = True
        for x in (self.k, self.v):
            x.masked_fill_(~used[:, None, :, None], NAN_CODE)
        for x in (self.ks, self.vs):
            x[~used.any(1)] = math.nan

    def cache(self, pkg, dev):
        return pkg.PagedKvCache.from_tensors(self.k.to(dev).view(torch.float8_e4m3fn),
                                             self.v.to(dev).view(torch.float8_e4m3fn), self.ks.to(dev), self.vs.to(dev))

    def batch(self, pkg, dev, **more):
        return pkg.PagedBatch(self.cu.to(dev), self.lens.to(dev), self.table.to(dev),
                              **{"max_q": self.max_q, "max_len": self.max_len, **more})


def attend64(c: Case, q: torch.Tensor, scale=D ** -0.5, window=0, sinks=0):
    """(out, lse, weighted size of the values, largest sum |q k|) in 64 bits; q [tokens][heads][128]."""
    t, heads, _ = q.shape
    group = heads // c.kv
    out, size = torch.zeros(t, heads, D, dtype=torch.float64), torch.zeros(t, heads, D, dtype=torch.float64)
    lse = torch.full((t, heads), -math.inf, dtype=torch.float64)
    reach = torch.zeros(t, heads, dtype=torch.float64)
    for b, (n_new, n) in enumerate(c.seqs):
        if n_new == 0 or n <= 0:
            continue
        rows = slice(int(c.cu[b]), int(c.cu[b + 1]))
        at = c.table[b, :-(-n // c.page)].long()
        inside = ((at >= 0) & (at < c.pages)).repeat_interleave(c.page)[:n]
        at = at.clamp(0, c.pages - 1)
        j, pos = torch.arange(n), torch.arange(n - n_new, n)
        sees = (j <= pos[:, None]) & inside & (pos >= 0)[:, None]
        if window > 0:
            sees &= (pos[:, None] - j < window) | (j < sinks)
        for h in range(heads):
            kv = h // group
            k = (code_values(c.k[at, kv]) * c.ks[at, kv].double()[:, None, None]).flatten(0, 1)[:n]
            v = (code_values(c.v[at, kv]) * c.vs[at, kv].double()[:, None, None]).flatten(0, 1)[:n]
            x = q[rows, h].double()
            s = torch.where(sees, x @ torch.nan_to_num(k).T * scale, torch.tensor(-math.inf, dtype=torch.float64))
            poisoned = (sees & k.isnan().any(1)).any(1)
            m = s.amax(1, keepdim=True).clamp_min(-1e300)
            e = torch.exp(s - m)
            z = e.sum(1, keepdim=True)
            w = e / z.clamp_min(1e-300)
            out[rows, h] = w @ torch.nan_to_num(v)
            size[rows, h] = w @ torch.nan_to_num(v).abs()
            lse[rows, h] = (m + z.log())[:, 0]
            reach[rows, h] = ((x.abs() @ torch.nan_to_num(k).abs().T) * abs(scale) * sees).amax(1)
            out[rows, h][poisoned] = math.nan
            lse[rows, h][poisoned] = math.nan
    return out, lse, size, reach


def attend_bounds(c: Case, out, size, reach, dtype):
    """Allowed distances of (out, lse) from 64 bits.  out: its own rounding; each probability rounded to f16
    (2^-11 of its share, or 2^-25 of the largest value's scale below f16's normal range) and off by
    the score's error; the score: 128 products summed in 32 bits, at most 2^-17 of the sum of their sizes."""
    unit = 2.0 ** -10 if dtype == torch.float16 else 2.0 ** -8
    score = reach[..., None] * 2.0 ** -17 + 2.0 ** -18
    vmax = 448.0 * float(torch.nan_to_num(c.vs).max())
    return unit * out.abs() + (2.0 ** -11 + 2 * score) * size + c.max_len * 2.0 ** -25 * vmax + 2.0 ** -24, score[..., 0]


def rope64(x: torch.Tensor, cos, sin, pos):
    half = cos.shape[1]
    y = x.double().clone()
    c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
    a, b = x[..., :half].double(), x[..., half:2 * half].double()
    y[..., :half], y[..., half:2 * half] = a * c - b * s, b * c + a * s
    return y


def append64(c: Case, k, v, cos, sin):
    """The cache after the append, as (values before rounding, scales, which slots are new, which tokens'
    heads are not finite, which slots hold nothing: past a sequence's end in a page that was written)
    for K and V.  Slots are [page][head][slot]."""
    res = []
    pos = torch.cat([torch.arange(n - q, n) for q, n in c.seqs]) if c.tokens else torch.zeros(0, dtype=torch.long)
    kx, vx = rope64(k, cos, sin, pos), v.double()
    bad = ~(kx.isfinite().all(-1) & vx.isfinite().all(-1))
    for codes, scales, x in ((c.k, c.ks, kx), (c.v, c.vs, vx)):
        val, sc = code_values(codes) * scales.double()[:, :, None, None], scales.double().clone()
        new = torch.zeros(c.pages, c.kv, c.page, dtype=torch.bool)
        broken, free = torch.zeros_like(new), torch.zeros_like(new)
        for b, (n_new, n) in enumerate(c.seqs):
            if n_new == 0:
                continue
            p0 = n - n_new
            for at in range(p0 // c.page, (n - 1) // c.page + 1):
                pid = int(c.table[b, at])
                if not 0 <= pid < c.pages:
                    continue
                lo, hi = max(p0, at * c.page), min(n, (at + 1) * c.page)
                rows = slice(int(c.cu[b]) + lo - p0, int(c.cu[b]) + hi - p0)
                for h in range(c.kv):
                    ok = ~bad[rows, h]
                    y = x[rows, h]
                    s = power_scale(float(y[ok].abs().max()) if ok.any() else 0.0)
                    if lo > at * c.page:
                        s = max(s, float(scales[pid, h]))
                    sc[pid, h] = s
                    val[pid, h, lo - at * c.page:hi - at * c.page] = y
                    free[pid, h, hi - at * c.page:] = True
                    new[pid, h, lo - at * c.page:hi - at * c.page] = True
                    broken[pid, h, lo - at * c.page:hi - at * c.page] = ~ok
        res.append((val, sc, new, broken, free))
    return res


def rope_tables(rope_dim: int, n: int):
    inv = 10000.0 ** (-torch.arange(0, rope_dim, 2, dtype=torch.float64) / max(rope_dim, 1))
    at = torch.arange(n, dtype=torch.float64)[:, None] * inv
    return at.cos().float(), at.sin().float()


def verify64(logits, cu, draft, u, noise, probs=None, temperature=None, max_q=None):
    """(tokens, accepted, logprobs, margin per sequence): the definition in 64 bits; margin is how near the
    closest decision of the sequence came to a tie, relative."""
    x, cu = np.asarray(logits, dtype=np.float64), np.asarray(cu)
    n, vocab = len(cu) - 1, x.shape[1]
    tokens, accepted = np.full((n, max_q), -1, dtype=np.int64), np.zeros(n, dtype=np.int64)
    logprobs, margin = np.zeros((n, max_q)), np.full(n, np.inf)
    for b in range(n):
        t0 = 1.0 if temperature is None else float(temperature[b])
        t = t0 or 1.0
        rows = int(cu[b + 1] - cu[b])
        if rows == 0:
            continue

        def row(i):
            l = x[cu[b] + i]
            if np.isnan(l).any() or (l == np.inf).any() or (l == -np.inf).all():
                return None, None
            z = l / t
            m = z.max()
            s = np.exp(z - m).sum()
            return np.exp(z - m) / s, (z - m) - np.log(s)

        i = 0
        while i < rows - 1:
            at = int(cu[b]) - b + i
            tok = int(draft[at])
            p, lp = row(i)
            if p is None or not 0 <= tok < vocab:
                break
            if t0 == 0:
                stands = int(np.argmax(x[cu[b] + i])) == tok
            else:
                q = 1.0 if probs is None else float(probs[at][tok])
                stands = float(u[at]) * q < p[tok]
                margin[b] = min(margin[b], abs(float(u[at]) * q - p[tok]) / max(p[tok], 1e-300))
            if not stands:
                break
            tokens[b, i], logprobs[b, i] = tok, lp[tok]
            i += 1
        accepted[b] = i
        p, lp = row(i)
        if p is None:
            continue
        if t0 == 0:
            tokens[b, i] = int(np.argmax(x[cu[b] + i]))
        else:
            r = p.copy()
            if i < rows - 1:
                at = int(cu[b]) - b + i
                if probs is not None:
                    r = np.maximum(p - np.asarray(probs[at], dtype=np.float64), 0)
                elif 0 <= int(draft[at]) < vocab:
                    r[int(draft[at])] = 0
                if not (r > 0).any():
                    r = p
            race = np.where(r > 0, r / np.asarray(noise[b], dtype=np.float64), -1.0)
            tokens[b, i] = int(np.argmax(race))
            two = np.sort(race)[-2:]
            if len(two) == 2 and two[0] > 0 and two[0] != two[1]:
                margin[b] = min(margin[b], (two[1] - two[0]) / two[1])
        logprobs[b, i] = lp[tokens[b, i]]
    return tokens, accepted, logprobs, margin
