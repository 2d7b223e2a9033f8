"""examples/speculative_decode.py: append, attention and verification together.  With temperature 0 drafted
decoding gives the tokens of decoding one by one, but for the rounding that the paths differ by."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest


def load():
    at = Path(__file__).resolve().parents[1] / "examples" / "speculative_decode.py"
    spec = importlib.util.spec_from_file_location("speculative_decode", at)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_lookup_drafts():
    ex = load()
    assert ex.lookup_drafts([1, 2, 3, 4, 1, 2], 2) == [3, 4]
    assert ex.lookup_drafts([1, 2, 3, 1, 2], 4) == [3, 1, 2, 2]
    assert ex.lookup_drafts([5, 6, 7], 2) == [7, 7]
    assert ex.lookup_drafts([5, 6, 7], 0) == []
    assert ex.lookup_drafts([9], 1) == [9]


@pytest.mark.gpu
def test_drafted_decoding_gives_the_tokens_of_plain_decoding(pkg, dev):
    import random
    ex = load()
    r = random.Random(3)
    prompts = [[r.randrange(2048) for _ in range(n)] for n in (17, 150, 70, 300)]
    plain, steps, _ = ex.generate(ex.Decoder(pkg, dev), prompts, 24, 0)
    drafted, fewer, stood = ex.generate(ex.Decoder(pkg, dev), prompts, 24, 4)
    assert steps == 24 and fewer <= steps and [len(t) for t in drafted] == [24] * 4
    # a near tie of two logits may fall either way and change what follows: at most one sequence here
    assert sum(a != b for a, b in zip(plain, drafted)) <= 1
    again, _, _ = ex.generate(ex.Decoder(pkg, dev), prompts, 24, 4)
    assert again == drafted
    sampled, _, _ = ex.generate(ex.Decoder(pkg, dev), prompts, 24, 3, temperature=0.8, seed=5)
    assert all(0 <= t < 2048 for line in sampled for t in line)
