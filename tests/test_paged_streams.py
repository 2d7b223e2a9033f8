"""Objects made on one stream, whose work is not done, and first used on another: what their constructors write is in
place before the first call."""
from __future__ import annotations

import numpy as np
import pytest
import torch
from paged_cases import D, Case, code_values, rope_tables, verify64
from test_verify_gpu import MARGIN, inputs

pytestmark = pytest.mark.gpu


@pytest.fixture
def busy(dev):
    """Keeps the current stream at work for some ten milliseconds."""
    big = torch.empty(1 << 28, device=dev)
    big.normal_()
    torch.cuda.synchronize()

    def go():
        for _ in range(20):
            big.normal_()
    return go


def test_verifier(pkg, dev, busy):
    vocab = 20011
    logits, cu, draft, u, noise, probs = inputs([3, 5, 2], vocab, 5)
    d = [torch.from_numpy(x).to(dev) if isinstance(x, np.ndarray) else x.to(dev) for x in (logits, cu, draft, u, noise, probs)]
    dirty = pkg.DraftVerifier(vocab, dev, max_seqs=3, max_rows=10, max_q=5)  # its memory is handed out again, not zero
    dirty.verify(*d[:5], draft_probs=d[5])  # (a kernel's first launch may wait for the device)
    dirty.ws.fill_(255), dirty.tokens.fill_(7)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    del dirty
    busy()
    ver = pkg.DraftVerifier(vocab, dev, max_seqs=3, max_rows=10, max_q=5)
    got = ver.verify(*d[:5], draft_probs=d[5], stream=stream)
    torch.cuda.synchronize()
    tokens, accepted, _, margin = verify64(logits.numpy(), cu, draft, u, noise, probs, None, 5)
    assert (margin > MARGIN).all()
    assert np.array_equal(got[0].cpu().numpy(), tokens) and np.array_equal(got[1].cpu().numpy(), accepted)


def test_cache(pkg, dev, busy):
    c = Case([(20, 20), (7, 7)], 16, 2, seed=3)
    k, v = c.randn(c.tokens, 2, D).to(dev), c.randn(c.tokens, 2, D).to(dev)
    cos, sin = (x.to(dev) for x in rope_tables(64, 32))
    batch = c.batch(pkg, dev)
    stream = torch.cuda.Stream()
    dirty = pkg.PagedKvCache(c.pages, dev, kv_heads=2, page_size=16)
    dirty.append(batch, None, k, v, cos, sin)  # (a kernel's first launch may wait for the device)
    torch.cuda.synchronize()
    del dirty
    busy()
    cache = pkg.PagedKvCache(c.pages, dev, kv_heads=2, page_size=16)
    cache.append(batch, None, k, v, cos, sin, stream=stream)
    torch.cuda.synchronize()
    at = c.table[1, 0].long()
    got = code_values(cache.v.view(torch.uint8)[at].cpu()) * cache.v_scale[at].cpu().double()[:, None, None]
    want = v[20:].cpu().double().transpose(0, 1)
    assert ((got[:, :7] - want).abs() <= 2.0 ** -4 * want.abs() + 2.0 ** -10).all()
