"""The workspace of PagedKvCache.attend: a call that needs a larger one must not take the old one from graphs that
were captured with it, and none is made inside a capture."""
from __future__ import annotations

import gc
import weakref

import pytest
import torch
from paged_cases import D, Case, attend64, attend_bounds


def test_a_replaced_workspace_stays(pkg):
    cache = pkg.PagedKvCache(2, "cpu", kv_heads=2, page_size=16)
    first = weakref.ref(cache.workspace(1, 1, 12))
    size = first().numel()
    assert cache.workspace(1, 500, 12).numel() > size
    gc.collect()
    assert first() is not None and not first().any()
    assert cache.workspace(1, 1, 12) is cache.workspace(1, 500, 12)


def test_status_is_that_of_every_workspace(pkg, monkeypatch):
    cache = pkg.PagedKvCache(2, "cpu", kv_heads=2, page_size=16)
    assert cache.status() == pkg.MMRS_OK
    first = cache.workspace(1, 1, 12).data_ptr()
    cache.workspace(1, 500, 12)
    real = pkg.lib()

    class Lib:
        def mmrs_paged_attend_status(self, ws):
            return pkg.MMRS_ERR_TIMEOUT if ws == first else pkg.MMRS_OK

        def __getattr__(self, name):
            return getattr(real, name)

    monkeypatch.setattr(pkg, "lib", Lib)
    assert cache.status() == pkg.MMRS_ERR_TIMEOUT


@pytest.mark.gpu
def test_replay_after_a_larger_call(pkg, dev):
    c = Case([(1, 900), (1, 500), (1, 33)], 64, 2, seed=8)
    q = c.randn(c.tokens, 12, D).to(torch.float16)
    ref, _, size, reach = attend64(c, q)
    bound, _ = attend_bounds(c, ref, size, reach, torch.float16)
    cache, batch, q_dev = c.cache(pkg, dev), c.batch(pkg, dev), q.to(dev)
    out = torch.empty_like(q_dev)
    cache.attend(batch, q_dev, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attend(batch, q_dev, out=out)
    # a prompt over the same cache, which needs more; then whatever memory is free is taken and filled
    long = Case([(300, 900)], 64, 2, seed=8)
    long.table = c.table[:1]
    cache.attend(long.batch(pkg, dev), long.randn(300, 12, D).half().to(dev))
    torch.cuda.synchronize()
    held = [torch.full((n,), 255, dtype=torch.uint8, device=dev) for n in (cache._spaces[0].numel(),) * 4]
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert ((out.cpu().double() - ref).abs() <= bound).all()
    assert all((h == 255).all() for h in held) and cache.status() == pkg.MMRS_OK


@pytest.mark.gpu
def test_no_workspace_is_made_inside_a_capture(pkg, dev):
    c = Case([(1, 90)], 64, 2, seed=2)
    q = c.randn(1, 12, D).to(torch.float16)
    cache, batch, q_dev = c.cache(pkg, dev), c.batch(pkg, dev), q.to(dev)
    out = torch.zeros_like(q_dev)
    with pytest.raises(pkg.MoeError, match="capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            cache.attend(batch, q_dev, out=out)
    torch.cuda.synchronize()
    cache.workspace(1, 1, 12)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attend(batch, q_dev, out=out)
    graph.replay()
    torch.cuda.synchronize()
    ref, _, size, reach = attend64(c, q)
    bound, _ = attend_bounds(c, ref, size, reach, torch.float16)
    assert ((out.cpu().double() - ref).abs() <= bound).all()
