"""How the prompt attention's softmax warps walk the pieces of their block when a bounded wait runs out: a model
on the CPU of the loop's control flow, with the rules read from the kernel's source.  (A wait that runs out is not
staged on a GPU.)  All eight warps have to reach the barriers of the cut items equally often, whatever warp fails
in whatever piece, or the block never ends."""
from __future__ import annotations

import random
import re
from pathlib import Path

SOURCE = Path(__file__).resolve().parents[1] / "minimax-rs_b200" / "csrc" / "paged_attend_prompt.cu"


def advances_when_failed() -> bool:
    """Whether a warp goes on to the next piece after its wait ran out (else it keeps the old one)."""
    cond = re.search(r"if \(([^{}]*?)\) \{?\s*pp_next\(p, sm, u \+ s\.n, u1, lane, next\)", SOURCE.read_text())
    assert cond, "the softmax loop's step to the next piece"
    return "ok" not in re.findall(r"\w+", cond.group(1))


def pieces(items, share, block):
    """(item, off, n) of the block's part of the list; items: tiles of each."""
    u, res = 0, []
    u0, u1 = share * block, min(share * (block + 1), sum(items))
    for at, nb in enumerate(items):
        lo, hi = max(u, u0), min(u + nb, u1)
        if lo < hi:
            res.append((at, lo - u, hi - lo))
        u += nb
    return res, u0, u1


def barriers(items, two_tiles, share, block, row_tile, fails_at, advance):
    """The items at whose barrier a warp arrives, in order; its wait runs out in its piece number `fails_at`."""
    todo, u, u1 = pieces(items, share, block)
    at, ok, seen = 0, True, []
    while u < u1:
        item, off, n = todo[at]
        mine = row_tile == 0 or two_tiles[item]
        c0, c1 = (u - off) // share, (u - off + items[item] - 1) // share
        if mine and fails_at is not None and at >= fails_at:
            ok = False
        if (ok or advance) and u + n < u1:
            at += 1
        if c0 != c1:
            seen.append(item)
        u += n
    return seen


def disagreements(advance, trials=400):
    r, bad = random.Random(5), 0
    for _ in range(trials):
        items = [r.randint(1, 12) for _ in range(r.randint(1, 30))]
        two = [r.random() < 0.6 for _ in items]
        blocks = r.randint(1, 12)
        share = max(1, -(-sum(items) // blocks))
        for block in range(-(-sum(items) // share)):
            n = len(pieces(items, share, block)[0])
            ways = {tuple(barriers(items, two, share, block, w >> 2, r.choice([None, r.randrange(n)]), advance))
                    for w in range(8)}
            bad += len(ways) > 1
    return bad


def test_the_model_tells_the_rules_apart():
    assert disagreements(advance=False) > 0


def test_every_warp_reaches_the_same_barriers_after_a_failed_wait():
    assert disagreements(advances_when_failed()) == 0


def counts_when_failed() -> bool:
    """Whether a block that gave up counts as arrived at the cut items it held a piece of."""
    rule = re.search(r"sm\.last = ([^;]*)atomicAdd\(p\.counters \+ c0, 1u\)", SOURCE.read_text())
    assert rule, "the block's arrival at a cut item"
    return "abort" not in rule.group(1)


def test_every_call_leaves_the_counters_at_zero():
    """An item's last block to arrive puts its counter back: so every block has to arrive, one that gave up, too.
    (The next call on the workspace would otherwise take an earlier block for the last and join too soon.)"""
    r, every = random.Random(6), counts_when_failed()
    for _ in range(200):
        items = [r.randint(1, 12) for _ in range(r.randint(1, 30))]
        share = max(1, -(-sum(items) // r.randint(1, 12)))
        blocks = -(-sum(items) // share)
        counters, failed = [0] * blocks, [r.random() < 0.3 for _ in range(blocks)]
        for block in r.sample(range(blocks), blocks):
            todo, u, _ = pieces(items, share, block)
            for item, off, n in todo:
                c0, c1 = (u - off) // share, (u - off + items[item] - 1) // share
                if c0 != c1 and (every or not failed[block]):
                    counters[c0] = 0 if counters[c0] == c1 - c0 else counters[c0] + 1
                u += n
        assert not any(counters)
