"""mmrs_verify_drafts_n: no draft past the given ones is read.  How many drafts the rows ask for is known on the
device only (sequences without rows bring none), so the arrays' length bounds the reads."""
from __future__ import annotations

import numpy as np
import pytest
import torch
from paged_cases import verify64
from test_verify_gpu import MARGIN, inputs

P = 1 << 20  # an address with every alignment; the checks come before any CUDA call


def args(**ch):
    a = dict(logits=P, type=0, vocab=1000, cu=P, num_seqs=4, rows=3, max_q=4, draft=P, probs=P, u=P, num_drafts=2, noise=P,
             temp=None, tokens=P, accepted=P, logprobs=P, ws=P, ws_bytes=1 << 40)
    a.update(ch)
    return (*a.values(), None)


@pytest.mark.parametrize("ch,name", [
    (dict(num_drafts=-1), "ARG"), (dict(draft=None), "ARG"), (dict(u=None), "ARG"), (dict(type=3), "UNSUPPORTED"),
    (dict(vocab=0), "ARG"), (dict(noise=None), "ARG"), (dict(ws=P + 16), "ARG"), (dict(ws_bytes=256), "ARG"),
])
def test_refusals(pkg, ch, name):
    assert pkg.lib().mmrs_verify_drafts_n(*args(**ch)) == getattr(pkg, "MMRS_ERR_" + name)


def test_nothing(pkg):
    assert pkg.lib().mmrs_verify_drafts_n(*args(num_seqs=0, rows=0, cu=None, num_drafts=0, draft=None, u=None)) == pkg.MMRS_OK


@pytest.mark.gpu
@pytest.mark.parametrize("with_probs", [True, False])
@pytest.mark.parametrize("temperature", [None, 0.0])
@pytest.mark.parametrize("rows_of,given", [([3, 2, 0, 0], 1), ([3, 0, 0, 0], 0), ([5, 4, 3, 0, 0, 0, 0], 5), ([4, 4], 6)])
def test_drafts_that_are_not_given_fall(pkg, dev, rows_of, given, temperature, with_probs):
    vocab, n, live = 3001, len(rows_of), [r for r in rows_of if r]
    logits, cu, draft, u, noise, probs = inputs(live, vocab, 7 * sum(rows_of) + given)
    cu = np.concatenate([cu, np.full(n - len(live), cu[-1], dtype=np.int32)])
    noise = np.concatenate([noise] + [noise[:1]] * (n - len(live)))
    draft[0::2] = logits.float().numpy().argmax(1)[[int(cu[b]) + i for b in range(len(live)) for i in range(live[b] - 1)]][0::2]
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    temp = None if temperature is None else np.full(n, temperature, dtype=np.float32)
    ver = pkg.DraftVerifier(vocab, dev, max_seqs=n, max_rows=sum(rows_of), max_q=max(rows_of))
    got = [x.cpu() for x in ver.verify(logits.to(dev), to(cu), to(draft[:given]), to(u[:given]), to(noise),
                                       draft_probs=to(probs[:given]) if with_probs else None,
                                       temperature=None if temp is None else to(temp))]
    # to the definition: a draft outside the vocabulary, of a model that gave nothing any probability
    draft[given:], probs[given:] = -1, 0.0
    tokens, accepted, _, margin = verify64(logits.float().numpy(), cu, draft, u, noise, probs if with_probs else None, temp,
                                           max(rows_of))
    sure = margin > MARGIN
    assert (~sure).sum() <= 1
    assert np.array_equal(got[1].numpy()[sure], accepted[sure]) and np.array_equal(got[0].numpy()[sure], tokens[sure])


@pytest.mark.gpu
def test_call_without_drafts(pkg, dev):
    """The entry point without a count: null arrays are no drafts, whatever rows a sequence has."""
    vocab = 1000
    logits, cu, _, _, noise, _ = inputs([3], vocab, 3)
    cu = np.concatenate([cu, [3, 3]]).astype(np.int32)
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    d_logits, d_cu, d_noise = logits.to(dev), to(cu), to(np.concatenate([noise] * 3))
    ver = pkg.DraftVerifier(vocab, dev, max_seqs=3, max_rows=3, max_q=3)
    rc = pkg.lib().mmrs_verify_drafts(d_logits.data_ptr(), 0, vocab, d_cu.data_ptr(), 3, 3, 3, None, None, None,
                                      d_noise.data_ptr(), None, *ver._ptrs, torch.cuda.current_stream().cuda_stream)
    assert rc == pkg.MMRS_OK
    tokens, accepted, _, margin = verify64(logits.float().numpy(), cu, np.full(2, -1), np.zeros(2), np.concatenate([noise] * 3),
                                           None, None, 3)
    assert margin[0] > MARGIN and np.array_equal(ver.tokens.cpu().numpy(), tokens)
    assert np.array_equal(ver.accepted.cpu().numpy(), accepted)
