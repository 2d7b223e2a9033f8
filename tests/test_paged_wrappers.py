"""Calls that the Python classes have to take: one token in a view of any row stride."""
from __future__ import annotations

import pytest
import torch
from paged_cases import D, Case, attend64, attend_bounds


@pytest.mark.parametrize("width", [12 * D, 12 * D + 3, 12 * D + 64])
def test_the_row_stride_of_one_token_does_not_matter(pkg, width):
    """The stride between rows is never used when there is one; the entry point asks for a multiple of eight."""
    one = torch.zeros(1, width, dtype=torch.float16).as_strided((1, 12, D), (width, D, 1))
    assert one.stride(0) == width
    assert pkg._tokens(one, None, "q") == (1, 12, 12 * D)
    assert pkg._tokens(one.expand(1, 12, D), 12, "q") == (1, 12, 12 * D)
    two = torch.zeros(2, width, dtype=torch.float16).as_strided((2, 12, D), (width, D, 1))
    assert pkg._tokens(two, None, "q") == (2, 12, width)


@pytest.mark.gpu
def test_one_token_of_an_odd_row_stride(pkg, dev):
    c = Case([(1, 300)], 64, 2, seed=1)
    wide = c.randn(1, 12 * D + 3).half()
    q = wide[:, :12 * D].unflatten(1, (12, D))
    q_dev = wide.to(dev).as_strided((1, 12, D), (12 * D + 3, D, 1))
    out = c.cache(pkg, dev).attend(c.batch(pkg, dev), q_dev)
    ref, _, size, reach = attend64(c, q)
    bound, _ = attend_bounds(c, ref, size, reach, torch.float16)
    assert ((out.cpu().double() - ref).abs() <= bound).all()
