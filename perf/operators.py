"""Cases of the paged decoding operators: appending rotated keys and values to a paged 8-bit cache,
attention over that cache, and the verification of drafted tokens.

A serving step with drafted tokens runs the three one after the other: the new tokens' keys and
values go into the cache, their queries read it, and the logits of the drafted positions decide how
many drafts stand.  `run` computes one of them in plain torch operations (32 bits, rounded once at
the end) or, where `own` is set, through minimax-rs_b200's public classes.

The cache holds e4m3 codes [pages][kv_heads][page_size][128] and one f32 scale (a power of two) per
page and head; a sequence's position j lies in slot j % page_size of page page_table[b][j // page_size].
"""
import math

import torch

own = False

D = 128  # head_dim
VOCAB = 200064  # MiniMax-M2.7's vocabulary
MAX_POS = 196608  # and its context
MIN_SCALE = 2.0 ** -64
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


# ---------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------
def listed():
    app = {"op": "append", "q_heads": 48, "kv_heads": 8, "rope_dim": 64}
    att = {"op": "attend", "q_heads": 48, "kv_heads": 8, "window": 0, "sinks": 0}
    ver = {"op": "verify", "vocab": VOCAB}
    return [
        # one user's next token: the smallest call, where the launch is what it costs
        dict(app, name="append 1x1", dtype="f16", page=64, seqs=1, q_lo=1, q_hi=1, len_lo=4001, len_hi=4001),
        # a batch of users, each with 4 drafted tokens and the last accepted one
        dict(app, name="append 64x5", dtype="bf16", page=64, seqs=64, q_lo=5, q_hi=5, len_lo=77, len_hi=3000),
        # ragged prompt chunks straight from f32 projections
        dict(app, name="append prompts", dtype="f32", page=32, seqs=6, q_lo=33, q_hi=4097, len_lo=4100, len_hi=6001),
        # one user's next token at a short context
        dict(att, name="attend 1x1 4k", dtype="f16", page=64, seqs=1, q_lo=1, q_hi=1, len_lo=4096, len_hi=4096),
        # one user's next token at the model's full context
        dict(att, name="attend 1x1 192k", dtype="f16", page=128, seqs=1, q_lo=1, q_hi=1, len_lo=MAX_POS, len_hi=MAX_POS),
        # the drafted tokens of a batch of users at ragged contexts
        dict(att, name="attend 64x5 ragged", dtype="bf16", page=64, seqs=64, q_lo=5, q_hi=5, len_lo=1001, len_hi=8192),
        # a sliding-window layer with visible first tokens, one rank of two, small pages
        dict(att, name="attend 48x1 window", dtype="f16", page=16, seqs=48, q_lo=1, q_hi=1, len_lo=700, len_hi=32768,
             q_heads=24, kv_heads=4, window=1024, sinks=4),
        # a prompt chunk behind a long prefix
        dict(att, name="attend prompt 4096", dtype="f16", page=64, seqs=1, q_lo=4096, q_hi=4096, len_lo=16384,
             len_hi=16384),
        # ragged prompts and single tokens in one call, windowed, eight query heads to a KV head
        dict(att, name="attend mixed window", dtype="bf16", page=32, seqs=5, q_lo=1, q_hi=2049, len_lo=2100, len_hi=7001,
             q_heads=32, kv_heads=4, window=511, sinks=16),
        # one user's four drafts
        dict(ver, name="verify 1x4", dtype="f32", seqs=1, d_lo=4, d_hi=4, probs=True),
        # a batch of users, four drafts each, with the draft model's probabilities
        dict(ver, name="verify 64x4", dtype="f32", seqs=64, d_lo=4, d_hi=4, probs=True),
        # drafts looked up in the text (no probabilities), ragged counts, bf16 logits
        dict(ver, name="verify 33 ragged", dtype="bf16", seqs=33, d_lo=0, d_hi=7, probs=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "verify"])
    if op == "verify":
        seqs = _log(rng, 1, 64)
        hi = rng.randint(1, 4 if seqs > 32 else 7)
        return {"op": op, "vocab": rng.choice([VOCAB, _log(rng, 1000, VOCAB)]), "dtype": rng.choice(["f32", "f16", "bf16"]),
                "seqs": seqs, "d_lo": rng.choice([hi, rng.randint(0, hi)]), "d_hi": hi, "probs": rng.random() < 0.6}
    group, kv = rng.choice([1, 2, 4, 5, 6, 6, 6, 8, 12, 16]), rng.choice([1, 2, 4, 8])
    c = {"op": op, "dtype": rng.choice(["f16", "bf16"]), "q_heads": group * kv, "kv_heads": kv,
         "page": rng.choice([16, 32, 64, 128])}
    if op == "append":
        c["dtype"] = rng.choice(["f16", "bf16", "f32"])
        c["rope_dim"] = rng.choice([0, 32, 64, 64, 128])
        c["seqs"] = _log(rng, 1, 64)
        hi = _log(rng, 1, max(8, min(4096, 16384 // c["seqs"])))
        c["q_lo"], c["q_hi"] = rng.choice([hi, rng.randint(1, hi)]), hi
        c["len_lo"] = hi + rng.randint(0, 500)
        c["len_hi"] = c["len_lo"] + rng.randint(0, 1500)
        return c
    c["window"] = rng.choice([0, 0, _log(rng, 1, 4096)])
    c["sinks"] = rng.choice([0, rng.randint(1, 64)]) if c["window"] else 0
    if rng.random() < 0.6:  # single tokens and drafts
        c["seqs"] = _log(rng, 1, 64)
        hi = rng.choice([1, 1, rng.randint(2, 8)])
        c["q_lo"], c["q_hi"] = rng.choice([hi, 1]), hi
        c["len_hi"] = _log(rng, 16, min(65536, 400000 // c["seqs"]))
    else:  # prompts
        c["seqs"] = rng.randint(1, 4)
        hi = _log(rng, 9, 2048)
        c["q_lo"], c["q_hi"] = rng.choice([hi, rng.randint(1, hi)]), hi
        c["len_hi"] = hi + _log(rng, 1, 6000)
    c["len_hi"] = max(c["len_hi"], c["q_hi"])
    c["len_lo"] = rng.choice([c["len_hi"], rng.randint(c["q_hi"], c["len_hi"])])
    return c


def _spread(lo, hi, n, step):
    """n whole numbers from lo to hi, in a scrambled order that the case alone decides."""
    if n == 1:
        return [hi]
    return [lo + (hi - lo) * ((i * step + 1) % n) // (n - 1) for i in range(n)]


def _coprime(n, at):
    return next(k for k in range(at, at + n + 1) if math.gcd(k, n) == 1)


def _lens(c):
    """(new tokens, positions after them) of every sequence."""
    n = c["seqs"]
    return _spread(c["q_lo"], c["q_hi"], n, _coprime(n, 3)), _spread(c["len_lo"], c["len_hi"], n, _coprime(n, 7))


def _visible(c, q, length):
    """(keys that some new token of a sequence sees, the sum over its tokens of the keys each sees)."""
    w, s, p0 = c["window"], c["sinks"], length - q
    if w <= 0:
        return length, sum(range(p0 + 1, length + 1))
    first = max(0, p0 - w + 1)
    seen = sum(min(p + 1, w) + min(s, max(0, p + 1 - w)) for p in range(p0, length))
    return length - first + min(s, first), seen


def work(case):
    c = case
    size = {"f32": 4, "f16": 2, "bf16": 2}[c["dtype"]]
    if c["op"] == "verify":
        drafts = sum(_spread(c["d_lo"], c["d_hi"], c["seqs"], _coprime(c["seqs"], 3)))
        rows = drafts + c["seqs"]
        some = c["seqs"] if drafts else 0
        nbytes = rows * c["vocab"] * size + c["seqs"] * c["vocab"] * 4 + (some * c["vocab"] * 4 if c["probs"] else 0)
        return {"bytes": nbytes + drafts * 8 + c["seqs"] * (4 + 8 * (c["d_hi"] + 1)), "flops": 4 * rows * c["vocab"]}
    qs, ls = _lens(c)
    t = sum(qs)
    if c["op"] == "append":
        pages = sum((n - 1) // c["page"] - (n - q) // c["page"] + 1 for q, n in zip(qs, ls))
        nbytes = t * c["q_heads"] * D * (size + 2) + 2 * t * c["kv_heads"] * D * (size + 1)
        return {"bytes": nbytes + pages * c["kv_heads"] * 8 + t * c["rope_dim"] * 4,
                "flops": 3 * t * (c["q_heads"] + c["kv_heads"]) * c["rope_dim"] + 2 * t * c["kv_heads"] * D}
    keys, seen = zip(*(_visible(c, q, n) for q, n in zip(qs, ls)))
    nbytes = sum(keys) * c["kv_heads"] * (2 * D + 8 / c["page"]) + t * c["q_heads"] * (2 * D * size + 4)
    return {"bytes": int(nbytes), "flops": 4 * D * c["q_heads"] * sum(seen)}


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------
def _scale_of(amax):
    """The smallest power of two s with amax <= 448 s, at least 2^-64; 0 where amax is 0."""
    m, e = torch.frexp(amax)  # 448 = 0.875 * 2^9
    s = torch.ldexp(torch.ones_like(amax), e - 9 + (m > 0.875).to(e.dtype)).clamp_min(MIN_SCALE)
    return torch.where(amax > 0, s, torch.zeros_like(s))


def _codes(x, scale):
    """e4m3 values of x / scale as bytes (a scale of 0 belongs to zeros)."""
    return (x / torch.where(scale > 0, scale, torch.ones_like(scale))).to(torch.float8_e4m3fn).view(torch.uint8)


def _pool(g, pages, kv_heads, page, level):
    """A cache half in use: normal values whose size differs by head and channel, quantised by page."""
    dev = g.device
    amp = level * torch.exp(0.4 * torch.randn(1, kv_heads, 1, D, generator=g, device=dev))
    x = torch.randn(pages, kv_heads, page, D, generator=g, device=dev).mul_(amp)
    scale = _scale_of(x.abs().amax((2, 3)))
    return _codes(x, scale[:, :, None, None]).view(torch.float8_e4m3fn), scale


def _rope_tables(rope_dim, n, dev):
    inv = 5e6 ** (-torch.arange(0, rope_dim, 2, device=dev, dtype=torch.float64) / max(rope_dim, 1))
    at = torch.arange(n, device=dev, dtype=torch.float64)[:, None] * inv
    return at.cos().float().contiguous(), at.sin().float().contiguous()


def _package():
    from __graft_entry__ import load_package
    return load_package()


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    dt = TYPES[c["dtype"]]
    s = {"op": c["op"], "case": c}
    if c["op"] == "verify":
        ds = _spread(c["d_lo"], c["d_hi"], c["seqs"], _coprime(c["seqs"], 3))
        n, v, drafts = c["seqs"], c["vocab"], sum(ds)
        rows = drafts + n
        # a model's logits: a broad floor, a few hundred plausible tokens, one or two that stand out
        logits = 2.0 * torch.randn(rows, v, generator=g, device=dev)
        top = (torch.randint(0, v, (rows, 1), generator=g, device=dev) + torch.arange(200, device=dev) * (v // 200)) % v
        logits.scatter_add_(1, top, 12.0 * torch.rand(rows, 200, generator=g, device=dev))
        logits = logits.to(dt)
        is_draft = torch.ones(rows, dtype=torch.bool, device=dev)
        is_draft[torch.tensor([sum(ds[:b + 1]) + b for b in range(n)], device=dev)] = False
        temp = 0.6 + 0.6 * torch.rand(n, generator=g, device=dev)
        temp[torch.arange(n, device=dev) % 8 == 5] = 0.0  # some users decode greedily
        row_t = torch.repeat_interleave(temp, torch.tensor([d + 1 for d in ds], device=dev))[is_draft]
        close = logits[is_draft].float() + 0.7 * torch.randn(drafts, v, generator=g, device=dev)
        q = torch.softmax(close / torch.where(row_t > 0, row_t, torch.ones_like(row_t))[:, None], -1)
        noise = torch.empty(drafts, v, device=dev).exponential_(1.0, generator=g)
        s["draft_tokens"] = (q / noise).argmax(-1).to(torch.int32)
        s["draft_probs"] = q if c["probs"] else None
        s["logits"], s["temperature"] = logits, temp
        s["uniforms"] = torch.rand(drafts, generator=g, device=dev)
        s["noise"] = torch.empty(n, v, device=dev).exponential_(1.0, generator=g).clamp_min_(1e-30)
        s["cu"] = ints([0] + [sum(ds[:b + 1]) + b + 1 for b in range(n)])
        s["max_q"] = max(ds) + 1
        if own:
            s["verifier"] = _package().DraftVerifier(v, dev, max_seqs=n, max_rows=rows, max_q=s["max_q"])
        return s
    qs, ls = _lens(c)
    page, t = c["page"], sum(qs)
    used = [-(-n // page) for n in ls]
    pages = sum(used) + 3
    perm = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.full((c["seqs"], max(used) + 1), -1, dtype=torch.int32, device=dev)
    for b, n in enumerate(used):
        table[b, :n] = perm[sum(used[:b]):sum(used[:b]) + n]
    s.update(cu=ints([0] + [sum(qs[:b + 1]) for b in range(c["seqs"])]), seq_len=ints(ls), table=table, max_q=max(qs),
             max_len=max(ls), page=page)
    s["k"], s["k_scale"] = _pool(g, pages, c["kv_heads"], page, 1.0)
    s["v"], s["v_scale"] = _pool(g, pages, c["kv_heads"], page, 0.5)
    if c["op"] == "append":
        # one projection's output, queries, keys and values side by side in each row
        width = (c["q_heads"] + 2 * c["kv_heads"]) * D
        qkv = torch.randn(t, width, generator=g, device=dev).mul_(torch.exp(
            0.4 * torch.randn(1, width, generator=g, device=dev))).to(dt)
        s["q"], s["k_new"], s["v_new"] = (x.unflatten(1, (-1, D)) for x in qkv.split(
            [c["q_heads"] * D, c["kv_heads"] * D, c["kv_heads"] * D], 1))
        s["cos"], s["sin"] = _rope_tables(c["rope_dim"], max(ls) + 1, dev)
        s["out"] = torch.empty(t, c["q_heads"], D, dtype=torch.bfloat16 if dt == torch.bfloat16 else torch.float16,
                               device=dev)
    else:
        s["q"] = (1.7 * torch.randn(t, c["q_heads"], D, generator=g, device=dev)).to(dt)
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(t, c["q_heads"], device=dev)
    if own:
        pkg = _package()
        s["cache"] = pkg.PagedKvCache.from_tensors(s["k"], s["v"], s["k_scale"], s["v_scale"])
        s["batch"] = pkg.PagedBatch(s["cu"], s["seq_len"], s["table"], max_q=s["max_q"], max_len=s["max_len"])
    return s


# ---------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------
def run(state):
    s = state
    if own:
        if s["op"] == "append":
            s["cache"].append(s["batch"], s["q"], s["k_new"], s["v_new"], s["cos"], s["sin"], q_out=s["out"])
            return {"q": s["out"], "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
        if s["op"] == "attend":
            s["cache"].attend(s["batch"], s["q"], window=s["case"]["window"], sinks=s["case"]["sinks"], out=s["out"],
                              lse=s["lse"])
            return {"out": s["out"], "lse": s["lse"]}
        tokens, accepted, logprobs = s["verifier"].verify(s["logits"], s["cu"], s["draft_tokens"], s["uniforms"],
                                                          s["noise"], draft_probs=s["draft_probs"],
                                                          temperature=s["temperature"])
        return {"tokens": tokens, "accepted": accepted, "logprobs": logprobs}
    return {"append": _append, "attend": _attend, "verify": _verify}[s["op"]](s)


def _token_index(s):
    """(sequence, index among its new tokens) of every new token."""
    cu = s["cu"].long()
    t = s["q"].shape[0]
    seq = torch.repeat_interleave(torch.arange(cu.numel() - 1, device=cu.device), cu.diff(), output_size=t)
    return seq, torch.arange(t, device=cu.device) - cu[seq]


def _rope(x, cos, sin, pos):
    """x [t][heads][128]: the pairs (i, i + rope_dim / 2) turned by the angle of their position."""
    h = cos.shape[1]
    a, b, rest = x[..., :h], x[..., h:2 * h], x[..., 2 * h:]
    c, n = cos[pos][:, None], sin[pos][:, None]
    return torch.cat([a * c - b * n, b * c + a * n, rest], -1)


def _store(pool, scales, x, pid, slot, seq, first_pid, first_slot):
    """Quantises x [t][heads][128] into the pool; a page that held tokens before keeps its scale or, where
    the new tokens need a larger one, has its older codes rounded again."""
    pages, heads, page, _ = pool.shape
    codes = pool.view(torch.uint8)
    amax = x.abs().amax(-1)
    need = torch.zeros(pages, heads, device=x.device).scatter_reduce_(0, pid[:, None].expand(-1, heads), amax, "amax")
    need = _scale_of(need)
    held = torch.zeros(pages, 1, dtype=torch.bool, device=x.device)
    held[first_pid, 0] = first_slot > 0
    touched = torch.zeros(pages, 1, dtype=torch.bool, device=x.device)
    touched[pid, 0] = True
    old = scales.clone()
    new = torch.where(touched, torch.where(held, torch.maximum(old, need), need), old)
    # the sequences' first pages: their older codes in the new scale
    ratio = old[first_pid] / torch.where(new[first_pid] > 0, new[first_pid], torch.ones_like(need[first_pid]))
    was = codes[first_pid]
    again = (was.view(torch.float8_e4m3fn).float() * ratio[:, :, None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    older = torch.arange(page, device=x.device)[None, None, :, None] < first_slot[:, None, None, None]
    codes[first_pid] = torch.where(older, again, was)
    codes[pid, :, slot] = _codes(x, new[pid][..., None])
    scales.copy_(new)


def _append(s):
    seq, i = _token_index(s)
    cu, page = s["cu"].long(), s["page"]
    start = s["seq_len"].long() - cu.diff()
    pos = start[seq] + i
    cos, sin = s["cos"], s["sin"]
    q = _rope(s["q"].float(), cos, sin, pos).to(s["out"].dtype)
    pid = s["table"].long()[seq, pos // page]
    slot = pos % page
    first = s["table"].long().gather(1, (start // page)[:, None])[:, 0]
    _store(s["k"], s["k_scale"], _rope(s["k_new"].float(), cos, sin, pos), pid, slot, seq, first, start % page)
    _store(s["v"], s["v_scale"], s["v_new"].float(), pid, slot, seq, first, start % page)
    return {"q": q, "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _gather(pool, scales, table):
    """[seqs][heads][positions][128] in 32 bits."""
    at = table.long().clamp_min(0)
    x = pool.view(torch.uint8)[at].view(torch.float8_e4m3fn).float() * scales[at][..., None, None]
    n, p, h, page, d = x.shape
    return x.transpose(1, 2).reshape(n, h, p * page, d)


def _attend(s):
    seq, i = _token_index(s)
    n, max_q, (t, heads, _) = s["cu"].numel() - 1, s["max_q"], s["q"].shape
    kv = s["k"].shape[1]
    group, dev = heads // kv, s["q"].device
    k, v = _gather(s["k"], s["k_scale"], s["table"]), _gather(s["v"], s["v_scale"], s["table"])
    q = torch.zeros(n, max_q, heads, D, device=dev)
    q[seq, i] = s["q"].float()
    q = q.view(n, max_q, kv, group, D).permute(0, 2, 1, 3, 4).reshape(n, kv, max_q * group, D)
    score = (q @ k.transpose(2, 3)).view(n, kv, max_q, group, -1).mul_(1.0 / math.sqrt(D))
    length = s["seq_len"].long()
    pos = (length - s["cu"].long().diff())[:, None] + torch.arange(max_q, device=dev)
    j = torch.arange(k.shape[2], device=dev)
    hidden = (j > pos[..., None]) | (j >= length[:, None, None])
    if s["case"]["window"] > 0:
        hidden |= (j <= pos[..., None] - s["case"]["window"]) & (j >= s["case"]["sinks"])
    score.masked_fill_(hidden[:, None, :, None, :], -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min(-3e38)
    e = score.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    o = (e.view(n, kv, max_q * group, -1) @ v).view(n, kv, max_q, group, D) / total.clamp_min(1e-38)
    lse = (top + total.log())[..., 0]
    pick = lambda x: x.transpose(1, 2)[seq, i].reshape(t, heads, *x.shape[4:])  # noqa: E731
    return {"out": pick(o).to(s["q"].dtype), "lse": pick(lse).contiguous()}


def _verify(s):
    cu, v, dev = s["cu"].long(), s["logits"].shape[1], s["logits"].device
    n, rows, most = cu.numel() - 1, s["logits"].shape[0], s["max_q"]
    seq = torch.repeat_interleave(torch.arange(n, device=dev), cu.diff(), output_size=rows)
    i = torch.arange(rows, device=dev) - cu[seq]
    count = cu.diff() - 1  # drafts
    greedy = s["temperature"] == 0
    temp = torch.where(greedy, torch.ones_like(s["temperature"]), s["temperature"])[seq]
    x = s["logits"].float() / temp[:, None]
    best = s["logits"].float().argmax(-1)
    top = x.amax(-1, keepdim=True)
    e = (x - top).exp()
    total = e.sum(-1, keepdim=True)
    p = e / total
    logp = lambda r, tok: (x[r, tok] - top[r, 0]) - total[r, 0].log()  # noqa: E731
    at = torch.arange(rows, device=dev)[i < count[seq]]  # the rows that judge a draft
    tok = s["draft_tokens"].long()
    q_tok = torch.ones(at.numel(), device=dev) if s["draft_probs"] is None else \
        s["draft_probs"].gather(1, tok[:, None])[:, 0]
    ok = torch.where(greedy[seq[at]], best[at] == tok, s["uniforms"] * q_tok < p[at, tok])
    stands = torch.zeros(n, most, dtype=torch.long, device=dev)
    stands[seq[at], i[at]] = ok.long()
    accepted = stands.cumprod(1).sum(1)
    row = cu[:-1] + accepted  # the row that gives the next token
    left = p[row]
    refused = accepted < count
    draft_row = (row - torch.arange(n, device=dev)).clamp(0, max(at.numel() - 1, 0))
    if at.numel() and s["draft_probs"] is not None:
        rest = (left - s["draft_probs"][draft_row]).clamp_min(0)
        left = torch.where((refused & (rest.amax(1) > 0))[:, None], rest, left)
    elif at.numel():
        rest = left.scatter(1, tok[draft_row][:, None], 0.0)
        left = torch.where((refused & (rest.amax(1) > 0))[:, None], rest, left)
    drawn = torch.where(left > 0, left / s["noise"], torch.full_like(left, -1.0)).argmax(-1)
    last = torch.where(greedy, best[row], drawn)
    tokens = torch.full((n, most), -1, dtype=torch.long, device=dev)
    tokens[seq[at], i[at]] = tok
    at_most = torch.arange(most, device=dev)[None]
    tokens = torch.where(at_most < accepted[:, None], tokens, torch.full_like(tokens, -1))
    tokens.scatter_(1, accepted[:, None], last[:, None])
    made = tokens >= 0
    lp = logp((cu[:-1, None] + at_most).clamp_max(rows - 1), tokens.clamp_min(0))
    return {"tokens": tokens.to(torch.int32), "accepted": accepted.to(torch.int32),
            "logprobs": torch.where(made, lp, torch.zeros_like(lp))}


# ---------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"append": _append64, "attend": _attend64, "verify": _verify64}[case["op"]](s)


def _append64(s):
    """What each stored code stands for, divided by its page's scale, before it is rounded to 8 bits."""
    cu, lens, page, half = s["cu"].tolist(), s["seq_len"].tolist(), s["page"], s["cos"].shape[1]
    out = {"q": s["q"].double(), "k": s["k"].double(), "v": s["v"].double(), "k_scale": s["k_scale"].double(),
           "v_scale": s["v_scale"].double()}
    k_new = s["k_new"].double()
    for b, n in enumerate(lens):
        p0 = n - (cu[b + 1] - cu[b])
        turn = torch.complex(s["cos"][p0:n].double(), s["sin"][p0:n].double())[:, None]
        for x in (out["q"], k_new):
            rows = x[cu[b]:cu[b + 1]]
            z = torch.complex(rows[..., :half].clone(), rows[..., half:2 * half].clone()) * turn
            rows[..., :half], rows[..., half:2 * half] = z.real, z.imag
    for name, x in (("k", k_new), ("v", s["v_new"].double())):
        pool, scale = out[name], out[name + "_scale"]
        for b, n in enumerate(lens):
            p0 = n - (cu[b + 1] - cu[b])
            for at in range(p0 // page, (n - 1) // page + 1):
                pid = int(s["table"][b, at])
                lo, hi = max(p0, at * page), min(n, (at + 1) * page)
                rows = x[cu[b] + lo - p0:cu[b] + hi - p0].transpose(0, 1)
                most = rows.abs().amax((1, 2))
                new = 2.0 ** (torch.floor(torch.log2(most)) - 8.0)
                new = torch.where(most > 448.0 * new, 2.0 * new, new).clamp_min(2.0 ** -64)
                if lo > at * page:
                    new = torch.maximum(new, scale[pid])
                    pool[pid, :, :lo - at * page] *= (scale[pid] / new)[:, None, None]
                pool[pid, :, lo - at * page:hi - at * page] = rows / new[:, None, None]
                scale[pid] = new
    return out


def _attend64(s):
    cu, lens, c = s["cu"].tolist(), s["seq_len"].tolist(), s["case"]
    page, kv, heads = s["page"], s["k"].shape[1], s["q"].shape[1]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    lse = torch.zeros(out.shape[:2], dtype=torch.float64, device=out.device)
    group = heads // kv
    for b, n in enumerate(lens):
        q = s["q"][cu[b]:cu[b + 1]].double()
        pids = s["table"][b, :-(-n // page)].long()
        pos = torch.arange(n - q.shape[0], n, device=q.device)[:, None]
        j = torch.arange(n, device=q.device)[None]
        sees = j <= pos
        if c["window"] > 0:
            sees &= (pos - j < c["window"]) | (j < c["sinks"])
        for h in range(kv):
            k = (s["k"][:, h].view(torch.uint8)[pids].view(torch.float8_e4m3fn).double()
                 * s["k_scale"][pids, h].double()[:, None, None]).flatten(0, 1)[:n]
            v = (s["v"][:, h].view(torch.uint8)[pids].view(torch.float8_e4m3fn).double()
                 * s["v_scale"][pids, h].double()[:, None, None]).flatten(0, 1)[:n]
            for g in range(h * group, (h + 1) * group):
                score = (q[:, g] @ k.T / math.sqrt(D)).masked_fill(~sees, -math.inf)
                z = torch.logsumexp(score, -1)
                out[cu[b]:cu[b + 1], g] = torch.exp(score - z[:, None]) @ v
                lse[cu[b]:cu[b + 1], g] = z
    return {"out": out, "lse": lse}


def _verify64(s):
    """The log-probabilities of the emitted tokens (whole numbers have no value in 64 bits of their own)."""
    plain = _verify(s)
    cu, tokens = s["cu"].tolist(), plain["tokens"].tolist()
    lp = torch.zeros(plain["logprobs"].shape, dtype=torch.float64)
    for b, line in enumerate(tokens):
        temp = float(s["temperature"][b]) or 1.0
        for i, tok in enumerate(line):
            if tok >= 0:
                lp[b, i] = torch.log_softmax(s["logits"][cu[b] + i].double() / temp, -1)[tok]
    return {"tokens": None, "accepted": None, "logprobs": lp}
