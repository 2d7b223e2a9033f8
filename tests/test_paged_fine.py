"""Paged attention within bounds that grow with a position's own weight (tests/paged_bounds.py): tight enough that
a value page that was left out, or read from elsewhere, fails at any length."""
from __future__ import annotations

import pytest
import torch
from paged_bounds import attend_fine, check_fine
from paged_cases import D, Case


@pytest.mark.parametrize("seqs,page", [([(1, 20000)], 64), ([(5, 9000)], 16), ([(130, 4100)], 64)])
def test_a_page_left_out_is_seen(seqs, page):
    """The bounds themselves: without the values of any one page, some row's error is at least twice what is allowed
    (so it is seen whatever the allowed error does)."""
    c = Case(seqs, page, 1, seed=1)
    q = (c.randn(c.tokens, 2, D) * 0.2).half()
    out, _, _, _, rms = attend_fine(c, q)
    pages = -(-seqs[0][1] // page)
    for at in [*range(0, pages, 7), pages - 1]:
        less = attend_fine(c, q, drop_page=(0, at))[0]
        assert ((less - out).square().mean(2).sqrt() > 2 * rms).any(), at


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", [0.2, 1.5])
@pytest.mark.parametrize("seqs,page", [([(1, 20000)], 64), ([(1, 20000), (1, 77), (1, 6000)], 128), ([(5, 9000)], 16),
                                       ([(3, 9000), (8, 1234)], 32), ([(130, 4100)], 64), ([(700, 700), (9, 2000)], 16)])
def test_long(pkg, dev, seqs, page, size, dtype):
    c = Case(seqs, page, 2, seed=seqs[0][1] + page)
    c.spoil_unused()
    c.vs.nan_to_num_(nan=2.0 ** -5), c.ks.nan_to_num_(nan=2.0 ** -5)  # (of pages that no sequence has)
    check_fine(pkg, dev, c, (c.randn(c.tokens, 12, D) * size).to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("group,kv", [(6, 2), (1, 3), (16, 1), (5, 2)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4), (17, 0)])
@pytest.mark.parametrize("seqs", [[(1, 1), (1, 2), (1, 300), (1, 1029)], [(5, 5), (2, 700), (8, 130)],
                                  [(1, 500), (5, 310), (300, 450), (0, 20), (17, 17)]])
def test_shapes(pkg, dev, seqs, group, kv, window, sinks):
    c = Case(seqs, 32, kv, seed=group + window)
    check_fine(pkg, dev, c, (c.randn(c.tokens, group * kv, D) * 0.7).half(), window=window, sinks=sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("group,kv", [(6, 2), (1, 2), (16, 1)])
@pytest.mark.parametrize("seqs", [[(5, 3), (1, 0), (2, 900), (8, 8)], [(60, 7), (300, 200), (3, 1)], [(1, 0)], [(70, 0)]])
def test_more_new_tokens_than_positions(pkg, dev, seqs, group, kv):
    """Rows before a sequence's first position see nothing: 0 and -infinity, next to rows that do."""
    c = Case(seqs, 16, kv, seed=group)
    c.max_len = max(c.max_len, 1)
    check_fine(pkg, dev, c, (c.randn(c.tokens, group * kv, D) * 0.7).half())
