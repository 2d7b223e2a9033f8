"""Draft verification on the GPU (mmrs_verify_drafts) against a plain 64-bit implementation
(tests/paged_cases.py: verify64).  A sequence whose closest decision lies within MARGIN of a tie in 64
bits is left out (32-bit exponentials are good to about 1e-6); at most a hundredth may be."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch
from paged_cases import verify64

pytestmark = pytest.mark.gpu
MARGIN = 1e-5


def inputs(rows_of, vocab, seed, dtype=torch.float32, sharp=3.0, near=0.6):
    """Logits, drafts drawn from a model near the target, its probabilities, and the random numbers."""
    g = np.random.default_rng(seed)
    n, rows = len(rows_of), sum(rows_of)
    cu = np.concatenate([[0], np.cumsum(rows_of)]).astype(np.int32)
    logits = torch.from_numpy((g.standard_normal((rows, vocab)) * sharp).astype(np.float32)).to(dtype)
    keep = [int(cu[b]) + i for b in range(n) for i in range(rows_of[b] - 1)]
    close = logits.float().numpy()[keep].astype(np.float64) + near * g.standard_normal((len(keep), vocab))
    p = np.exp(close - close.max(1, keepdims=True)) if keep else close
    probs = (p / p.sum(1, keepdims=True)).astype(np.float32) if keep else p.astype(np.float32)
    draft = np.array([g.choice(vocab, p=x.astype(np.float64) / x.astype(np.float64).sum()) for x in probs], dtype=np.int32)
    u = g.random(len(keep)).astype(np.float32)
    noise = np.maximum(g.exponential(size=(n, vocab)), 1e-30).astype(np.float32)
    return logits, cu, draft, u, noise, probs


def check(pkg, dev, args, probs, temperature, allow=0.01):
    logits, cu, draft, u, noise = args
    n, max_q = len(cu) - 1, int(np.diff(cu).max())
    ver = pkg.DraftVerifier(logits.shape[1], dev, max_seqs=n, max_rows=max(logits.shape[0], 1), max_q=max_q)
    to = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    call = lambda: ver.verify(logits.to(dev), to(cu), to(draft), to(u), to(noise), draft_probs=to(probs),  # noqa: E731
                              temperature=to(temperature))
    got = [x.cpu().clone() for x in call()]
    status = ver.status()
    again = [x.cpu() for x in call()]
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    tokens, accepted, logprobs, margin = verify64(logits.float().numpy(), cu, draft, u, noise, probs, temperature, max_q)
    sure = margin > MARGIN
    assert (~sure).sum() <= max(1, allow * n)
    assert np.array_equal(got[1].numpy()[sure], accepted[sure])
    assert np.array_equal(got[0].numpy()[sure], tokens[sure])
    # x - max and ln sum: two 32-bit differences of numbers up to |x| and a sum of exponentials good to 1e-6
    size = np.abs(np.nan_to_num(logits.float().numpy(), nan=0, posinf=0, neginf=0)).max()
    t = 1.0 if temperature is None else min([x for x in temperature if x > 0] + [1.0])
    assert np.abs(got[2].numpy() - logprobs)[sure].max() <= 4e-6 + 2.0 ** -21 * size / t
    bad = [b for b in range(n) if cu[b + 1] > cu[b] and sure[b] and tokens[b][accepted[b]] < 0]
    assert status == (pkg.MMRS_ERR_NONFINITE if bad else pkg.MMRS_OK) or not sure.all()
    return tokens, accepted


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("with_probs", [True, False])
@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 4099, 50001])
def test_small(pkg, dev, dtype, with_probs, vocab):
    rows = [5, 1, 3, 2, 8, 4]
    *args, probs = inputs(rows, vocab, vocab, dtype)
    temp = np.array([1.0, 0.7, 0.0, 1.3, 0.9, 0.0], dtype=np.float32)
    check(pkg, dev, args, probs if with_probs else None, temp)


@pytest.mark.parametrize("n,k", [(1, 5), (3, 2), (40, 3)])
def test_full_vocabulary(pkg, dev, n, k):
    *args, probs = inputs([k] * n, 200064, n, sharp=4.0)
    _, accepted = check(pkg, dev, args, probs, None)
    assert n < 40 or 0 < accepted.mean() < k - 1


def test_accepts_and_refuses_in_proportion(pkg, dev):
    """Over many draws the emitted first token follows the target's probabilities, whatever the draft's."""
    vocab, n = 6, 1000
    g = np.random.default_rng(2)
    row = np.array([1.0, 0.3, -0.4, 0.8, -2.0, 0.0], dtype=np.float32)
    q = np.array([0.05, 0.5, 0.05, 0.1, 0.2, 0.1], dtype=np.float32)
    args = (torch.from_numpy(np.tile(row, (2 * n, 1))), np.arange(0, 2 * n + 1, 2, dtype=np.int32),
            g.choice(vocab, size=n, p=q.astype(np.float64) / q.sum()).astype(np.int32), g.random(n).astype(np.float32),
            g.exponential(size=(n, vocab)).astype(np.float32))
    tokens, _ = check(pkg, dev, args, np.tile(q, (n, 1)), None)
    p = np.exp(row.astype(np.float64))
    p /= p.sum()
    count = np.bincount(tokens[:, 0], minlength=vocab)
    assert (np.abs(count - n * p) <= 5 * np.sqrt(n * p * (1 - p))).all()


@pytest.mark.parametrize("temp", [None, 0.0])
def test_ties_go_to_the_lowest_index(pkg, dev, temp):
    vocab = 3000
    logits = torch.zeros(4, vocab)
    logits[:, [700, 900, 2999]] = 5.0
    noise = np.full((2, vocab), 0.5, dtype=np.float32)
    args = (logits, np.array([0, 2, 4], dtype=np.int32), np.array([700, 900], dtype=np.int32),
            np.array([0.9999, 0.9999], dtype=np.float32), noise)
    t = None if temp is None else np.full(2, temp, dtype=np.float32)
    tokens, accepted = check(pkg, dev, args, None, t)
    assert accepted.tolist() == ([0, 0] if temp is None else [1, 0])
    assert tokens[:, 0].tolist() == ([900, 700] if temp is None else [700, 700])


def test_masked_and_broken_rows(pkg, dev):
    vocab = 1025
    *args, probs = inputs([3, 3, 3, 3, 3, 2, 1], vocab, 5)
    logits = args[0]
    logits[:, 500:] = -math.inf  # a mask that leaves the drafts of the upper half no chance
    logits[3] = -math.inf        # sequence 1: its first row has nothing
    logits[7, 3] = math.nan      # sequence 2
    logits[9, 4] = math.inf      # sequence 3
    logits[12:15] = -math.inf
    logits[12:15, 17] = -3.0     # sequence 4: one token left in each row
    args[2][8:10] = 17
    t = np.array([1, 1, 0, 1, 1, 0, 1], dtype=np.float32)
    tokens, accepted = check(pkg, dev, args, probs, t)
    assert tokens[1].tolist() == [-1, -1, -1] and tokens[3, 0] == -1 and tokens[4].tolist() == [17, 17, 17]
    t[:] = 0
    check(pkg, dev, args, probs, t)


def test_drafts_outside_the_vocabulary_and_certain_draws(pkg, dev):
    vocab = 777
    *args, probs = inputs([4, 4, 4], vocab, 11)
    args[2][0], args[2][4] = -1, vocab
    args[3][:] = 0.0  # u = 0: a draft of any probability stands
    check(pkg, dev, args, probs, None)
    check(pkg, dev, args, None, None)


def test_residual_nowhere_positive_falls_back_to_the_target(pkg, dev):
    vocab = 100
    *args, _ = inputs([2, 2], vocab, 13)
    probs = np.ones((2, vocab), dtype=np.float32)  # not a distribution: p - q < 0 everywhere
    args[3][:] = 0.999
    _, accepted = check(pkg, dev, args, probs, None)
    assert accepted.tolist() == [0, 0]


def test_sequences_without_rows_come_last(pkg, dev):
    *args, probs = inputs([3, 2], 500, 17)
    logits, cu, draft, u, noise = args
    cu = np.concatenate([cu, [5, 5]]).astype(np.int32)
    noise = np.concatenate([noise, noise])
    tokens, accepted = check(pkg, dev, (logits, cu, draft, u, noise), probs, None)
    assert (tokens[2:] == -1).all() and (accepted[2:] == 0).all()


def test_logits_beyond_the_range_of_exp(pkg, dev):
    *args, probs = inputs([3, 3, 3], 2000, 19, sharp=3.0)
    args[0].mul_(1e4)
    check(pkg, dev, args, probs, np.array([1.0, 50.0, 0.0], dtype=np.float32))


def test_another_stream_and_graph_replay(pkg, dev):
    logits, cu, draft, u, noise, probs = inputs([3, 4], 3000, 23)
    d = [torch.from_numpy(x).to(dev) if isinstance(x, np.ndarray) else x.to(dev) for x in (logits, cu, draft, u, noise, probs)]
    ver = pkg.DraftVerifier(3000, dev, max_seqs=2, max_rows=7, max_q=4)
    want = [x.cpu().clone() for x in ver.verify(*d[:5], draft_probs=d[5])]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    ver.tokens.fill_(5)
    torch.cuda.synchronize()
    ver.verify(*d[:5], draft_probs=d[5], stream=stream)
    stream.synchronize()
    assert torch.equal(ver.tokens.cpu(), want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ver.verify(*d[:5], draft_probs=d[5])
    for _ in range(3):
        ver.tokens.fill_(5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ver.tokens.cpu(), want[0]) and torch.equal(ver.accepted.cpu(), want[1])
