"""Serving several sequences with drafted tokens over a paged 8-bit cache.

    python examples/speculative_decode.py [--seqs 4] [--new 48] [--drafts 4] [--temperature 0.8]

A two-layer decoder of random weights with MiniMax's attention geometry (48 query heads, 8 KV heads of
128, 64 rotated columns) and small other sizes.  Prompts of different lengths go through in one call;
then every step appends each sequence's last token and its drafts (PagedKvCache.append), attends all of
them in one call (PagedKvCache.attend) and lets the target's logits decide how many drafts stand and
what comes next (DraftVerifier.verify).  Nothing is read back inside a step but the accepted tokens,
which the drafting (a lookup of the last two tokens in the sequence's own text) needs on the host.
"""
from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

HEADS, KV_HEADS, D, ROPE = 48, 8, 128, 64


class Decoder:
    """Random weights; each layer: norm, fused q/k/v projection, append + attend, output projection, and a
    plain two-matrix block."""

    def __init__(self, pkg, dev, hidden=512, layers=2, vocab=2048, max_len=4096, pages=256, page_size=64, seed=0):
        import torch
        self.pkg, self.torch, self.dev, self.vocab, self.page_size = pkg, torch, dev, vocab, page_size
        g = torch.Generator(device=dev).manual_seed(seed)
        w = lambda n, k, s=1.0: (torch.randn(n, k, generator=g, device=dev) * s / k ** 0.5).half()  # noqa: E731
        self.embed = torch.randn(vocab, hidden, generator=g, device=dev).half()
        self.layers = [dict(qkv=w((HEADS + 2 * KV_HEADS) * D, hidden, 2.0), out=w(hidden, HEADS * D, 2.0), up=w(4 * hidden, hidden),
                            down=w(hidden, 4 * hidden)) for _ in range(layers)]
        self.head = w(vocab, hidden, 6.0)
        self.caches = [pkg.PagedKvCache(pages, dev, kv_heads=KV_HEADS, page_size=page_size) for _ in range(layers)]
        inv = 5e6 ** (-torch.arange(0, ROPE, 2, device=dev, dtype=torch.float64) / ROPE)
        at = torch.arange(max_len, device=dev, dtype=torch.float64)[:, None] * inv
        self.cos, self.sin = at.cos().float().contiguous(), at.sin().float().contiguous()

    def logits(self, tokens, batch):
        """Logits [tokens][vocab] of the batch's new tokens (int64 [tokens])."""
        torch = self.torch
        norm = lambda x: x * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6).half()  # noqa: E731
        x = self.embed[tokens]
        for layer, cache in zip(self.layers, self.caches):
            qkv = (norm(x) @ layer["qkv"].T).unflatten(1, (-1, D))
            q, k, v = qkv.split([HEADS, KV_HEADS, KV_HEADS], 1)
            q = cache.append(batch, q, k, v, self.cos, self.sin)
            x = x + cache.attend(batch, q).flatten(1) @ layer["out"].T
            x = x + torch.nn.functional.silu(norm(x) @ layer["up"].T) @ layer["down"].T
        return (norm(x) @ self.head.T).float()


def lookup_drafts(text, count):
    """The tokens that followed the last two tokens where the text had them before (else its last ones)."""
    pair = text[-2:]
    for i in range(len(text) - 3, 0, -1):
        if text[i - 1:i + 1] == pair:
            found = text[i + 1:i + 1 + count]
            return found + text[-1:] * (count - len(found))
    return text[-1:] * count


def generate(model, prompts, new, drafts, temperature=0.0, seed=0):
    """`new` tokens for every prompt (lists of ids) with `drafts` drafted tokens a step (0: one by one).
    Returns (texts without the prompts, steps, drafts that stood)."""
    torch, pkg, dev = model.torch, model.pkg, model.dev
    n, page = len(prompts), model.page_size
    texts = [list(p) for p in prompts]
    longest = max(map(len, prompts)) + new + drafts + 2
    per_seq = -(-longest // page)
    table = torch.arange(n * per_seq, dtype=torch.int32, device=dev).view(n, per_seq)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    width = drafts + 1
    verifier = pkg.DraftVerifier(model.vocab, dev, max_seqs=n, max_rows=n * width, max_q=width)
    g = torch.Generator(device=dev).manual_seed(seed)
    temp = torch.full((n,), float(temperature), device=dev)

    # the prompts but for their last tokens, all in one call
    lens = [len(p) - 1 for p in prompts]
    cu = ints([0] + [sum(lens[:b + 1]) for b in range(n)])
    model.logits(torch.tensor([t for p in prompts for t in p[:-1]], device=dev),
                 pkg.PagedBatch(cu, ints(lens), table, max_q=max(lens), max_len=longest))
    # then steps of the last token and the drafts: one batch object, its lengths updated in place
    cu = ints([b * width for b in range(n + 1)])
    seq_len = ints([0] * n)
    batch = pkg.PagedBatch(cu, seq_len, table, max_q=width, max_len=longest)
    steps = stood = 0
    while min(len(t) - len(p) for t, p in zip(texts, prompts)) < new:
        live = [min(len(t), len(p) + new) for t, p in zip(texts, prompts)]
        texts = [t[:k] for t, k in zip(texts, live)]
        guess = [lookup_drafts(t, drafts) for t in texts]
        seq_len.copy_(ints([len(t) + drafts for t in texts]))
        logits = model.logits(torch.tensor([x for t, d in zip(texts, guess) for x in [t[-1]] + d], device=dev), batch)
        noise = torch.empty(n, model.vocab, device=dev).exponential_(1.0, generator=g).clamp_min_(1e-30)
        uniforms = torch.rand(n * drafts, generator=g, device=dev)
        tokens, accepted, _ = verifier.verify(logits, cu, ints([x for d in guess for x in d]), uniforms, noise,
                                              temperature=temp)
        for b, (line, k) in enumerate(zip(tokens.tolist(), accepted.tolist())):
            if len(texts[b]) < len(prompts[b]) + new:
                texts[b] += line[:k + 1]
                stood += k
        steps += 1
    assert verifier.status() == pkg.MMRS_OK and all(c.status() == pkg.MMRS_OK for c in model.caches)
    return [t[len(p):len(p) + new] for t, p in zip(texts, prompts)], steps, stood


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--seqs", type=int, default=4)
    ap.add_argument("--new", type=int, default=48)
    ap.add_argument("--drafts", type=int, default=4)
    ap.add_argument("--temperature", type=float, default=0.0)
    a = ap.parse_args()
    import random

    import torch
    from __graft_entry__ import load_package
    model = Decoder(load_package(), torch.device("cuda:0"))
    r = random.Random(1)
    prompts = [[r.randrange(model.vocab) for _ in range(r.randint(20, 400))] for _ in range(a.seqs)]
    for drafts in (0, a.drafts):
        torch.cuda.synchronize()
        t = time.perf_counter()
        texts, steps, stood = generate(model, prompts, a.new, drafts, a.temperature)
        torch.cuda.synchronize()
        print(f"{drafts} drafts a step: {a.new} tokens for {a.seqs} sequences in {steps} steps, {stood} drafts stood, "
              f"{time.perf_counter() - t:.3f} s; first: {texts[0][:12]}")


if __name__ == "__main__":
    main()
