"""Pages whose value scales lie far apart.  A page with large values need not have any weight in a row to be among
the positions that the kernels go through: the values of the others must not be lost next to it."""
from __future__ import annotations

import pytest
import torch
from paged_bounds import attend_fine, check_fine
from paged_cases import D, Case

pytestmark = pytest.mark.gpu


def far_apart(seqs, page, kv, drop, big, seed, level=0):
    """A case whose pages have values of size 2^level, but where big(page of a table) says so 2^drop times that;
    keys there point away from every query."""
    c = Case(seqs, page, kv, seed=seed)
    c.vs[:] = 2.0 ** (level - 5)
    c.ks[:] = 2.0 ** -6
    for b, (_, n) in enumerate(seqs):
        for at in range(-(-n // page)):
            if big(at):
                pid = int(c.table[b, at])
                c.vs[pid] = 2.0 ** (level - 5 + drop)
                c.ks[pid] = 2.0 ** -4
                c.k[pid, :, :, 0] = 0xFE  # -448
    return c


def queries(c, heads, dtype, away=True):
    q = c.randn(c.tokens, heads, D) * 0.5
    if away:
        q[..., 0] = 64.0  # 64 * 448 / 16 / sqrt 128 = 158 below the others
    return q.to(dtype)


@pytest.mark.parametrize("page", [16, 32, 128])
@pytest.mark.parametrize("drop", [10, 16, 20, 30, 60])
@pytest.mark.parametrize("group,kv,seqs", [(6, 4, [(1, 9000)] * 6), (4, 2, [(4, 7000)] * 8), (6, 2, [(4, 7000), (1, 500)] * 6),
                                           (6, 2, [(5, 500), (8, 640)])])
def test_tokens_and_drafts(pkg, dev, group, kv, seqs, drop, page):
    """Long enough that each warp of the kernel goes through several steps of both kinds."""
    c = far_apart(seqs, page, kv, drop, lambda at: at % 3 == 1, seed=drop + page)
    check_fine(pkg, dev, c, queries(c, kv * group, torch.bfloat16))


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("drop", [24, 60])
def test_rows_that_do_not_see_the_large_page(pkg, dev, drop, page):
    """The last page is large and only the last drafts see it; the first page is and a window hides it from some."""
    c = far_apart([(8, 10 * page + 3), (5, 20 * page + 2)] * 30, page, 2, drop, lambda at: at in (10, 20), seed=drop)
    check_fine(pkg, dev, c, queries(c, 12, torch.bfloat16, away=False))
    c = far_apart([(8, page + 60)] * 60, page, 2, drop, lambda at: at == 0, seed=drop)
    check_fine(pkg, dev, c, queries(c, 12, torch.bfloat16, away=False), window=63)


def test_values_down_to_the_smallest_scale(pkg, dev):
    """2^-64, the least that the append writes, next to 2^60."""
    c = far_apart([(1, 9000), (4, 5000)] * 6, 32, 2, 119, lambda at: at % 3 == 1, seed=3, level=-59)
    q = queries(c, 12, torch.bfloat16)
    cache = c.cache(pkg, dev)
    got = cache.attend(c.batch(pkg, dev), q.to(dev)).cpu().double()
    out, _, allow, _, _ = attend_fine(c, q)
    # (the bounds' smallest terms are far above these values: the error is taken relative to the outputs' size)
    size = out.square().mean().sqrt()
    assert (got - out).square().mean().sqrt() <= 2.0 ** -8 * size


def test_zero_scales_between(pkg, dev):
    c = far_apart([(1, 9000), (6, 7000)] * 6, 32, 2, 40, lambda at: at % 3 == 1, seed=4)
    for b in range(12):
        c.vs[c.table[b, 2].long()] = 0.0
        c.vs[c.table[b, 5].long()] = 0.0
    check_fine(pkg, dev, c, queries(c, 12, torch.float16))


PROMPTS = [(6, 2, [(300, 9000)] * 4), (1, 2, [(257, 5000), (60, 4000)] * 3), (8, 1, [(2000, 2100)]), (6, 2, [(130, 130), (9, 700)])]


@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("drop", [16, 24, 40, 80])
@pytest.mark.parametrize("group,kv,seqs", PROMPTS)
def test_prompts(pkg, dev, group, kv, seqs, drop, page):
    """Every third run of 128 positions is large."""
    c = far_apart(seqs, page, kv, drop, lambda at: at * page // 128 % 3 == 1, seed=drop + page)
    check_fine(pkg, dev, c, queries(c, kv * group, torch.bfloat16))


@pytest.mark.parametrize("page", [16, 32])
@pytest.mark.parametrize("drop", [14, 20])
@pytest.mark.parametrize("group,kv,seqs", PROMPTS)
def test_prompts_within_128_positions(pkg, dev, group, kv, seqs, drop, page):
    c = far_apart(seqs, page, kv, drop, lambda at: at % 3 == 1, seed=drop + page)
    check_fine(pkg, dev, c, queries(c, kv * group, torch.bfloat16))


@pytest.mark.parametrize("drop", [30, 60])
def test_prompt_rows_that_do_not_see_the_large_values(pkg, dev, drop):
    """The last 128 positions are large and only the last rows see them; then the first 128, behind a window."""
    c = far_apart([(300, 1280), (700, 900)], 64, 2, drop, lambda at: at in (18, 19), seed=drop)
    check_fine(pkg, dev, c, queries(c, 12, torch.bfloat16, away=False))
    c = far_apart([(500, 500), (120, 250)], 64, 2, drop, lambda at: at < 2, seed=drop)
    check_fine(pkg, dev, c, queries(c, 12, torch.bfloat16, away=False), window=40)


def test_prompts_with_zero_scales_between(pkg, dev):
    c = far_apart([(300, 3000), (100, 1500)], 64, 2, 40, lambda at: at // 2 % 3 == 1, seed=4)
    for b in range(2):
        for at in (0, 1, 4, 9):
            c.vs[c.table[b, at].long()] = 0.0
    check_fine(pkg, dev, c, queries(c, 12, torch.float16))
