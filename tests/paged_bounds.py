"""How far attention over the paged cache may be from 64 bits, position by position.

A weight w of a row is rounded on its way to the second product: by 2^-11 of itself, or, where its exponential
lies below f16's normal range (relative to the largest one of its block so far, which is at most the row's
largest), by 2^-25 of the row's largest weight 1 / Z; never by more than w.  Single tokens and drafts multiply
it, before that product, by the value scale of its page relative to a reference that is at most 2^6 times
as large: the second term grows by that ratio.  Prompts multiply the values instead: exact to 2^-22 of the
largest scale of the same 128 positions, below that to 2^-24 of it (half a unit of f16's smallest, 2^-25,
for a reference 2^7 below the largest and up to 2^8 off it).  A score is a sum of 128 products in 32 bits (at
most 2^-17 of the sum of their sizes), an exponential good to 2^-18.  The second product sums 16 positions
at a time in 32 bits.  At last the output is rounded to its own type.

Those are limits of each element.  They grow with the number of positions as if all roundings had one sign; over
the 128 elements of a row they do not, and the row's root mean square error is held to FACTOR times what
independent roundings give (each uniform: its limit / sqrt 3; the scores' 128 products at 2^-21 of their size
each), with the sums' error added as it is.  A row of 128 strays from its expectation by some 6 %; the factor of 4
leaves room for errors that go together within a row."""
from __future__ import annotations

import math

import torch
from paged_cases import D, Case, code_values

RATIO = 2.0 ** 6
FEW_ROWS = 48  # of a KV head: up to these a sequence counts as single tokens or drafts
FACTOR = 4.0


def attend_fine(c: Case, q: torch.Tensor, scale=D ** -0.5, window=0, sinks=0, drop_page=None):
    """(out, lse, allowed distance of out, of lse, allowed root mean square of a row of out) in 64 bits for finite
    caches and queries; q [tokens][heads][128].  drop_page: (sequence, page of its table) whose values count as zero in `out`."""
    t, heads, _ = q.shape
    group = heads // c.kv
    unit = 2.0 ** -11 if q.dtype == torch.float16 else 2.0 ** -8
    out, allow = (torch.zeros(t, heads, D, dtype=torch.float64) for _ in range(2))
    lse = torch.full((t, heads), -math.inf, dtype=torch.float64)
    lse_allow, rms = (torch.zeros(t, heads, dtype=torch.float64) for _ in range(2))
    for b, (n_new, n) in enumerate(c.seqs):
        if n_new == 0 or n <= 0:
            continue
        rows = slice(int(c.cu[b]), int(c.cu[b + 1]))
        prompt = n_new * group > FEW_ROWS
        at = c.table[b, :-(-n // c.page)].long()
        inside = ((at >= 0) & (at < c.pages)).repeat_interleave(c.page)[:n]
        at = at.clamp(0, c.pages - 1)
        j, pos = torch.arange(n), torch.arange(n - n_new, n)
        sees = (j <= pos[:, None]) & inside & (pos >= 0)[:, None]
        if window > 0:
            sees &= (pos[:, None] - j < window) | (j < sinks)
        for kv in range(c.kv):
            k = (code_values(c.k[at, kv]) * c.ks[at, kv].double()[:, None, None]).flatten(0, 1)[:n]
            vs = c.vs[at, kv].double().repeat_interleave(c.page)[:n]
            v = code_values(c.v[at, kv]).flatten(0, 1)[:n] * vs[:, None]
            v = torch.where(inside[:, None], v, torch.zeros_like(v))
            vs = torch.where(inside, vs, torch.zeros_like(vs))
            ratio = (vs.max() / vs.clamp_min(1e-300)).clamp_max(0.0 if prompt else RATIO)
            tile = torch.stack([x.max() for x in vs.split(128)]).repeat_interleave(128)[:n]
            kept = v.clone()
            if drop_page is not None and drop_page[0] == b:
                kept[drop_page[1] * c.page:(drop_page[1] + 1) * c.page] = 0
            for h in range(kv * group, (kv + 1) * group):
                x = q[rows, h].double()
                s = (x @ torch.nan_to_num(k).T * scale).masked_fill(~sees, -math.inf)
                m = s.amax(1, keepdim=True).clamp_min(-1e300)
                z = torch.exp(s - m).sum(1, keepdim=True)
                w = torch.exp(s - m) / z.clamp_min(1e-300)
                reach = ((x.abs() @ torch.nan_to_num(k).abs().T) * abs(scale) * sees).amax(1, keepdim=True)
                off = reach * 2.0 ** -17 + 2.0 ** -18
                sums = (n / 16 + 64) * 2.0 ** -23
                tail = torch.minimum(w, 2.0 ** -25 * (1 + ratio) / z.clamp_min(1.0))
                err = (2.0 ** -11 + 2 * off + sums) * w + tail
                out[rows, h] = w @ kept
                each = (2.0 ** -11 * w + tail) / 3 ** 0.5 + w * (reach * 2.0 ** -21 + 2.0 ** -18)
                square = each ** 2 @ v ** 2 + (unit * out[rows, h]) ** 2 / 3 + 2.0 ** -50
                walk = (w ** 2 @ v ** 2).mean(1).sqrt() + out[rows, h].square().mean(1).sqrt()
                rms[rows, h] = FACTOR * square.mean(1).sqrt() + sums * walk
                low = torch.minimum(v.abs(), (2.0 ** -24 * tile)[:, None]) * (prompt & (vs < 2.0 ** -22 * tile))[:, None]
                allow[rows, h] = err @ v.abs() + w @ low
                rms[rows, h] += (w @ low).square().mean(1).sqrt()
                lse[rows, h] = (m + z.log())[:, 0]
                lse_allow[rows, h] = off[:, 0] + sums + 2.0 ** -22 * lse[rows, h].abs().nan_to_num(posinf=0.0)
    return out, lse, allow * (1 + unit) + unit * out.abs() + 2.0 ** -25, lse_allow, rms


def check_fine(pkg, dev, c: Case, q: torch.Tensor, scale=None, window=0, sinks=0):
    """PagedKvCache.attend of the case within these bounds."""
    cache, batch = c.cache(pkg, dev), c.batch(pkg, dev)
    got_lse = torch.full(q.shape[:2], 7.0, device=dev)
    got = cache.attend(batch, q.to(dev), window=window, sinks=sinks, lse=got_lse, scale=scale).cpu().double()
    assert cache.status() == pkg.MMRS_OK
    out, lse, allow, lse_allow, rms = attend_fine(c, q, D ** -0.5 if scale is None else scale, window, sinks)
    got_lse = got_lse.cpu().double()
    empty = lse == -math.inf
    assert torch.equal(got_lse == -math.inf, empty) and (got[empty] == 0).all()
    live = ~empty
    assert ((got_lse - lse).abs() <= lse_allow)[live].all()
    off = (got - out).abs()
    assert (off <= allow)[live].all(), float((off / allow)[live].max())
    off = (got - out).square().mean(2).sqrt()
    assert (off <= rms)[live].all(), float((off / rms)[live].max())
