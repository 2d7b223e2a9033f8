"""One DraftVerifier for batches of any size up to its own: users come and go, and a batch that shrinks may
grow again.  Each call against the 64-bit definition (tests/paged_cases.py: verify64)."""
from __future__ import annotations

import numpy as np
import pytest
import torch
from paged_cases import verify64
from test_verify_gpu import MARGIN, inputs

# (test_verify_gpu.inputs is pure numpy; the marks below are this module's own)


def test_no_call_moves_what_is_kept_between_calls(pkg):
    """The records' counters must stay zero from one call to the next, so nothing that a call writes may lie
    where a call of another size has its records: the place of the parts is the same for all of them.
    Their beginning is the workspace's size less the parts', which are as many as the rows."""
    need = pkg.lib().mmrs_verify_workspace_bytes
    per_row = need(1, 2) - need(1, 1)
    begins = {need(n, rows) - rows * per_row for n in (0, 1, 2, 8, 64, 1024) for rows in (0, 1, 5, 320, 65536)}
    assert len(begins) == 1, begins


def call(pkg, dev, ver, rows_of, vocab, seed, temperature, dtype=torch.float32):
    logits, cu, draft, u, noise, probs = inputs(rows_of, vocab, seed, dtype)
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    n = len(rows_of)
    temp = None if temperature is None else np.full(n, temperature, dtype=np.float32)
    ver.tokens.fill_(-7)  # a call that writes nothing must not pass with the last one's tokens
    ver.accepted.fill_(-7)
    got = [x.cpu().clone() for x in ver.verify(logits.to(dev), to(cu), to(draft), to(u), to(noise), draft_probs=to(probs),
                                               temperature=None if temp is None else to(temp))]
    assert ver.status() == pkg.MMRS_OK
    tokens, accepted, _, margin = verify64(logits.float().numpy(), cu, draft, u, noise, probs, temp, ver.max_q)
    sure = margin > MARGIN
    assert (~sure).sum() <= 1
    assert np.array_equal(got[1].numpy()[sure], accepted[sure]), rows_of
    assert np.array_equal(got[0].numpy()[sure], tokens[sure]), rows_of


@pytest.mark.gpu
@pytest.mark.parametrize("temperature", [None, 0.0])
@pytest.mark.parametrize("sizes", [(8, 1, 8), (3, 2, 8), (8, 1, 2, 3, 8)])
def test_batches_that_shrink_and_grow(pkg, dev, sizes, temperature):
    vocab = 200064
    ver = pkg.DraftVerifier(vocab, dev, max_seqs=8, max_rows=40, max_q=5)
    for at, n in enumerate(sizes):
        call(pkg, dev, ver, [5] * n, vocab, 31 * at + n, temperature)


@pytest.mark.gpu
def test_greedy_then_sampled_of_other_types_and_sizes(pkg, dev):
    vocab = 50001
    ver = pkg.DraftVerifier(vocab, dev, max_seqs=40, max_rows=160, max_q=5)
    for at, (n, t, dtype) in enumerate([(2, 0.0, torch.float32), (40, None, torch.bfloat16), (1, 0.7, torch.float16),
                                        (17, 0.0, torch.float16), (5, None, torch.float32), (40, 0.9, torch.float32)]):
        call(pkg, dev, ver, [1 + (3 * b + at) % 4 for b in range(n)], vocab, at, t, dtype)
